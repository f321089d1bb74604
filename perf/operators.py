"""The cache operators of gofann on a GPU: what is timed, on which inputs, and their plain forms.

A language model's key/value cache is a vector store that every new token searches.  The operators are

  append   new rows are rotated by their positions (rotary embedding, both layouts, part of the head) and keys and
           values are written to a paged cache in 4 bits; the 8-bit bounds of the touched blocks are renewed
  select   an int8 upper bound of q.k over each block of 64 cached tokens picks the blocks that a query reads
  attend   attention of the query rows over the 4-bit cache: over all of it (causal, windowed, filtered by a bit per
           token) or over the selected blocks

A page holds 64 tokens.  The chunk of one (page, key/value head) of a head_dim D (64 or 128, G = D / 64 groups) is

  key codes     [kt 4][grp G][g1 4][g0 2][t 4][j 4][e 2][r 2] bytes, low nibble n = 0, high nibble n = 1:
                token 16 g1 + 4 kt + 2 r + g0, dimension 64 grp + 16 t + 4 j + 2 n + e
  key params    [g1 4][g0 2][kt 4][r 2][grp G] pairs of f16 (scale, minimum) of the token above
  value codes   [dt D/16][g 8][t 4][kt 4][e 2][r 2] bytes: dimension 16 dt + 8 r + g, token 16 t + 4 kt + 2 n + e
  value params  as the key params

and the value of a code c is c * scale + minimum.  The bounds of a (page, head) are int8 [2][D], the largest and the
smallest key value of each dimension in units of an f32 scale.
"""
import math
import os
import sys

import torch

own = False

PAGE, GROUP = 64, 64
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
CLAMP = 57344.0  # largest magnitude that the cache holds


# ------------------------------------------------------------------ the cases
def listed():
    append = dict(op="append", rotary=128, interleaved=False)
    select = dict(op="select", first=1, recent=2)
    attend = dict(op="attend", causal=True, window=0, n_select=0, bits=False)
    return [
        # one new token of one short conversation: launch latency
        dict(append, name="append one token", seqs=1, rows=1, ctx=1000, ragged=0, heads=32, kv_heads=8, dim=128,
             dtype="bf16"),
        # a decode step of a full serving batch, half of the head rotated
        dict(append, name="append a batch", seqs=96, rows=1, ctx=4001, ragged=37, heads=24, kv_heads=4, dim=128,
             dtype="f16", rotary=64),
        # chunks of five prompts, odd lengths that start and end inside pages
        dict(append, name="append prompts", seqs=5, rows=2043, ctx=9001, ragged=611, heads=32, kv_heads=8, dim=64,
             dtype="bf16", rotary=64, interleaved=True),
        # one query against the blocks of one long document
        dict(select, name="select for one token", seqs=1, rows=1, ctx=32700, ragged=0, heads=32, kv_heads=8, dim=128,
             dtype="bf16", n_select=32),
        # a decode step of 64 long conversations
        dict(select, name="select for a batch", seqs=64, rows=1, ctx=131072, ragged=1009, heads=32, kv_heads=4,
             dim=128, dtype="bf16", n_select=64),
        # every token of a prompt's chunk selects for itself
        dict(select, name="select for a chunk", seqs=1, rows=2043, ctx=40003, ragged=0, heads=16, kv_heads=2, dim=128,
             dtype="f16", n_select=48),
        # one token, short conversation: launch latency
        dict(attend, name="attend one token", seqs=1, rows=1, ctx=777, ragged=0, heads=32, kv_heads=8, dim=128,
             dtype="bf16"),
        # one token over one long document: the long axis is split
        dict(attend, name="attend a long document", seqs=1, rows=1, ctx=131072, ragged=0, heads=32, kv_heads=8,
             dim=128, dtype="bf16"),
        # a decode step of 32 conversations of uneven lengths
        dict(attend, name="attend a batch", seqs=32, rows=1, ctx=32768, ragged=701, heads=64, kv_heads=8, dim=128,
             dtype="bf16"),
        # chunks of two prompts over their own history
        dict(attend, name="attend prompts", seqs=2, rows=2043, ctx=12289, ragged=1999, heads=32, kv_heads=8, dim=128,
             dtype="bf16"),
        # a decode step over selected blocks, with evicted tokens
        dict(attend, name="attend selected blocks", seqs=48, rows=1, ctx=65536, ragged=907, heads=32, kv_heads=8,
             dim=128, dtype="bf16", n_select=64, bits=True),
        # a chunk whose tokens each read their own blocks
        dict(attend, name="attend selected, chunk", seqs=1, rows=509, ctx=20011, ragged=0, heads=32, kv_heads=4,
             dim=64, dtype="f16", n_select=32),
    ]


def log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(("append", "select", "attend", "attend"))
        kv_heads = rng.choice((1, 2, 4, 8))
        dim = rng.choice((64, 128, 128))
        case = dict(op=op, seqs=log_int(rng, 1, 96), rows=rng.choice((1, 1, 1, rng.randint(2, 8), log_int(rng, 9, 2048))),
                    ctx=log_int(rng, 1, 131072), ragged=rng.randint(0, 1500), heads=kv_heads * rng.choice((1, 2, 3, 4, 6, 8)),
                    kv_heads=kv_heads, dim=dim, dtype=rng.choice(("bf16", "bf16", "f16")))
        case["ctx"] = max(case["ctx"], case["rows"])
        blocks = -(-case["ctx"] // PAGE)
        if op == "append":
            case.update(rotary=rng.choice((0, dim // 2, dim, 2 * rng.randint(1, dim // 2))),
                        interleaved=rng.random() < 0.5)
        elif op == "select":
            case.update(n_select=rng.randint(2, 128), first=rng.randint(0, 1), recent=rng.randint(0, 1))
        else:
            case.update(causal=rng.random() < 0.8, window=rng.choice((0, 0, 0, log_int(rng, 16, 8192))),
                        n_select=rng.choice((0, 0, rng.randint(1, 64))), bits=rng.random() < 0.4)
        n_rows, pages = sum(rows_of(case)), case["seqs"] * blocks
        if pages * kv_heads * dim > 20e6 or n_rows > 12000:
            continue
        if op == "select" and n_rows * case["heads"] * blocks > 50e6:
            continue
        if op == "attend" and case["n_select"] and n_rows * kv_heads * min(case["n_select"], blocks) * dim > 17e6:
            continue
        if op == "attend" and not case["n_select"] and (case["seqs"] * case["rows"] * case["heads"] * blocks * PAGE > 1.5e9):
            continue
        return case


def lens_of(case):
    """Tokens of each sequence, this call's rows among them."""
    span = max(1, case["ctx"] - case["rows"] + 1)
    return [case["ctx"] - (s * case["ragged"]) % span for s in range(case["seqs"])]


def rows_of(case):
    """Query rows of each sequence: at most case["rows"]."""
    return [max(1, case["rows"] - (s * 13) % max(1, case["rows"] // 2)) for s in range(case["seqs"])]


def chunk_bytes(dim):
    return 64 * dim + 2 * 256 * (dim // GROUP)


def visible(case, length, rows):
    """Keys that each row of a sequence sees (every token of its cache counted as present)."""
    got = []
    for i in range(rows):
        end = length - rows + i + 1 if case["causal"] else length
        got.append(min(end, case["window"]) if case["window"] else end)
    return got


def work(case):
    lens, rows, d = lens_of(case), rows_of(case), case["dim"]
    h, kv, n = case["heads"], case["kv_heads"], sum(rows_of(case))
    pages = [-(-x // PAGE) for x in lens]
    bounds = 2 * d + 4
    if case["op"] == "append":
        per = d // 2 + 4 * (d // GROUP)  # one token's key or value in 4 bits
        touched = sum(-(-x // PAGE) - (x - r) // PAGE for x, r in zip(lens, rows))
        old = sum((x - r) % PAGE for x, r in zip(lens, rows))
        data = n * (2 * (2 * h + 4 * kv) * d + 4 * case["rotary"] + 2 * kv * per) + kv * (touched * bounds + old * per)
        return {"bytes": data, "flops": n * (h + kv) * 3 * case["rotary"] + n * kv * 2 * d * 6}
    if case["op"] == "select":
        data = sum(pages) * kv * bounds + n * (2 * h * d + 8 * kv * case["n_select"])
        return {"bytes": data, "flops": sum(r * p for r, p in zip(rows, pages)) * h * 4 * d}
    io = n * h * (4 * d + 4)
    if case["n_select"]:
        keys = [min(case["n_select"], p) * PAGE for p in pages]
        cache = sum(min(p, r * k // PAGE) for p, r, k in zip(pages, rows, keys)) * kv * chunk_bytes(d)
        ids = 4 * n * kv * case["n_select"]
        return {"bytes": cache + io + ids, "flops": sum(r * min(k, x) for r, k, x in zip(rows, keys, lens)) * h * 4 * d}
    seen = [visible(case, x, r) for x, r in zip(lens, rows)]
    reach = [min(p, -(-(max(v) + len(v)) // PAGE) + 1) if case["window"] else p for p, v in zip(pages, seen)]
    bits = sum(pages) * 8 if case["bits"] else 0
    return {"bytes": sum(reach) * kv * chunk_bytes(d) + io + bits, "flops": sum(map(sum, seen)) * h * 4 * d}


# ------------------------------------------------------------------ the inputs
def rotary_tables(length, rotary, base=10000.0):
    """cos and sin of position times frequency, from 64 bits."""
    f = base ** (-torch.arange(0, rotary, 2, device="cuda", dtype=torch.float64) / max(rotary, 1))
    a = torch.arange(length, device="cuda", dtype=torch.float64)[:, None] * f
    return a.cos().float(), a.sin().float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    def ints(lo, hi, shape, dtype):
        return torch.randint(lo, hi, shape, device="cuda", generator=g, dtype=dtype)

    lens, rows = lens_of(case), rows_of(case)
    d, kv, h, seqs = case["dim"], case["kv_heads"], case["heads"], case["seqs"]
    dtype, n = DTYPES[case["dtype"]], sum(rows)
    max_pages = max(-(-x // PAGE) for x in lens)
    n_pages = seqs * max_pages + 3
    s = dict(case=case, n_rows=n, max_rows=max(rows))
    s["page_table"] = torch.randperm(n_pages, device="cuda", generator=g)[: seqs * max_pages].reshape(seqs, max_pages).int()
    s["seq_len"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    offset = torch.zeros(seqs + 1, dtype=torch.int64)
    offset[1:] = torch.cumsum(torch.tensor(rows), 0)
    s["row_offset"] = offset.int().cuda()
    s["row_seq"] = torch.repeat_interleave(torch.arange(seqs), torch.tensor(rows)).cuda()
    s["row_pos"] = (torch.arange(n) - offset[:-1].repeat_interleave(torch.tensor(rows)) +
                    (torch.tensor(lens) - torch.tensor(rows)).repeat_interleave(torch.tensor(rows))).cuda()
    # one row of a fused projection: queries, keys and values next to each other
    fused = (normal(n, (h + 2 * kv) * d) * 1.5).to(dtype)
    s["q"] = fused[:, : h * d].unflatten(1, (h, d))
    s["k"] = fused[:, h * d : (h + kv) * d].unflatten(1, (kv, d))
    s["v"] = fused[:, (h + kv) * d :].unflatten(1, (kv, d))
    if case["op"] != "select":
        pages = ints(0, 256, (n_pages, kv, chunk_bytes(d)), torch.uint8)
        for at in (32 * d, 64 * d + 256 * (d // GROUP)):
            scale = torch.rand(n_pages, kv, 64 * (d // GROUP), device="cuda", generator=g) * 0.3 + 0.05
            low = scale * (torch.rand(scale.shape, device="cuda", generator=g) - 8.0)
            pages[..., at : at + 256 * (d // GROUP)] = torch.stack((scale, low), -1).half().view(torch.uint8).reshape(n_pages, kv, -1)
        s["pages"] = pages
    if case["op"] != "attend":
        middle = normal(n_pages, kv, 1, d) * 25
        half = normal(n_pages, kv, 1, d).abs() * 20 + 10
        s["bounds"] = torch.cat((middle + half, middle - half), 2).round().clamp(-127, 127).to(torch.int8)
        s["bound_scale"] = torch.rand(n_pages, kv, device="cuda", generator=g) * 0.02 + 0.01
    if case["op"] == "append":
        s["cos"], s["sin"] = rotary_tables(max(lens), case["rotary"])
        touched = [(i, b) for i, (x, r) in enumerate(zip(lens, rows)) for b in range((x - r) // PAGE, -(-x // PAGE))]
        s["touched"] = torch.tensor(touched, device="cuda")
        first, last = {}, 0
        for k, (i, _) in enumerate(touched):
            first.setdefault(i, k)
        first = torch.tensor([first[i] for i in range(seqs)], device="cuda")
        start = (torch.tensor(lens) - torch.tensor(rows)).cuda()
        s["row_touched"] = first[s["row_seq"]] + s["row_pos"] // PAGE - (start // PAGE)[s["row_seq"]]
    if case["op"] == "attend":
        s["scale"] = 1.0 / math.sqrt(d)
        if case["n_select"]:
            # distinct blocks of each row's past, the first and the newest among them, ascending, -1 at the end
            n_blocks = s["row_pos"][:, None] // PAGE + 1
            score = torch.rand(n, kv, max_pages, device="cuda", generator=g)
            at = torch.arange(max_pages, device="cuda")
            score = torch.where((at == 0) | (at == n_blocks[:, :, None] - 1), 2.0, score)
            score = torch.where(at < n_blocks[:, :, None], score, -1.0)
            k = min(case["n_select"], max_pages)
            top, ids = torch.topk(score, k, dim=-1)
            ids = torch.where(top < 0, max_pages, ids).sort(-1).values
            ids = torch.where(ids == max_pages, -1, ids)
            s["selected"] = torch.nn.functional.pad(ids, (0, case["n_select"] - k), value=-1).int()
        if case["bits"]:
            s["key_bits"] = ints(-(1 << 31), 1 << 31, (seqs, 2 * max_pages), torch.int64).int() | ints(-(1 << 31), 1 << 31, (seqs, 2 * max_pages), torch.int64).int()
    if own:
        package = os.path.join(os.getcwd(), "go-fann_b200")
        if package not in sys.path:
            sys.path.insert(0, package)
        from gofann import kv_cache

        s["cache"] = kv_cache.KVCache(d, pages=s.get("pages"), bounds=s.get("bounds"), bound_scale=s.get("bound_scale"))
        s["batch"] = kv_cache.KVBatch(s["page_table"], s["seq_len"], s["row_offset"], n, max(rows))
        if case["op"] == "append":
            s["out"] = (torch.empty(n, h, d, dtype=dtype, device="cuda"), torch.empty(n, kv, d, dtype=dtype, device="cuda"),
                        torch.empty(n, kv, d, dtype=dtype, device="cuda"))
        elif case["op"] == "select":
            s["out"] = (torch.empty(n, kv, case["n_select"], dtype=torch.int32, device="cuda"),
                        torch.empty(n, kv, case["n_select"], device="cuda"))
        else:
            s["out"] = (torch.empty(n, h, d, dtype=dtype, device="cuda"), torch.empty(n, h, device="cuda"))
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    if own:
        if case["op"] == "append":
            q_out, k_out, v_out = s["cache"].append(s["batch"], s["q"], s["k"], s["v"], cos=s["cos"], sin=s["sin"],
                                                    rotary_dim=case["rotary"], interleaved=case["interleaved"],
                                                    q_out=s["out"][0], k_out=s["out"][1], v_out=s["out"][2])
            return q_out, k_out, v_out, s["bounds"], s["bound_scale"]
        if case["op"] == "select":
            return s["cache"].select(s["batch"], s["q"], case["n_select"], first=case["first"], recent=case["recent"],
                                     ids=s["out"][0], scores=s["out"][1])
        return s["cache"].attend(s["batch"], s["q"], scale=s["scale"], causal=case["causal"], window=case["window"],
                                 selected=s.get("selected"), key_bits=s.get("key_bits"), out=s["out"][0], lse=s["out"][1])
    return {"append": plain_append, "select": plain_select, "attend": plain_attend}[case["op"]](s)


def key_codes(chunks, d):
    """[..., tokens 64, D] codes of the key half of chunks."""
    c = chunks[..., : 32 * d].unflatten(-1, (4, d // GROUP, 4, 2, 4, 4, 2, 2))
    c = torch.stack((c & 15, c >> 4), -1)  # kt grp g1 g0 t j e r n
    a = c.dim() - 9
    c = c.permute(*range(a), *(a + i for i in (2, 0, 7, 3, 1, 4, 5, 8, 6)))
    return c.reshape(*c.shape[:a], PAGE, d)


def value_codes(chunks, d):
    at = 32 * d + 256 * (d // GROUP)
    c = chunks[..., at : at + 32 * d].unflatten(-1, (d // 16, 8, 4, 4, 2, 2))
    c = torch.stack((c & 15, c >> 4), -1)  # dt g t kt e r n
    a = c.dim() - 7
    c = c.permute(*range(a), *(a + i for i in (2, 3, 6, 4, 0, 5, 1)))
    return c.reshape(*c.shape[:a], PAGE, d)


def params(chunks, d, at):
    """[..., tokens 64, G, 2] scale and minimum in 32 bits."""
    g = d // GROUP
    p = chunks[..., at : at + 256 * g].contiguous().view(torch.float16).unflatten(-1, (4, 2, 4, 2, g, 2))
    a = p.dim() - 6
    p = p.permute(*range(a), *(a + i for i in (0, 2, 3, 1, 4, 5)))
    return p.reshape(*p.shape[:a], PAGE, g, 2).float()


def values_of(codes, p):
    c = codes.unflatten(-1, (-1, GROUP)).float()
    return (c * p[..., 0:1] + p[..., 1:2]).flatten(-2)


def keys_and_values(chunks, d):
    k = values_of(key_codes(chunks, d), params(chunks, d, 32 * d))
    return k, values_of(value_codes(chunks, d), params(chunks, d, 64 * d + 256 * (d // GROUP)))


def pack(kc, kp, vc, vp, d):
    """The chunks of codes [..., 64, D] and of f16 params [..., 64, G, 2]."""
    g, lead = d // GROUP, kc.shape[:-2]
    a = len(lead)
    k = kc.reshape(*lead, 4, 4, 2, 2, g, 4, 4, 2, 2)  # g1 kt r g0 grp t j n e
    k = k.permute(*range(a), *(a + i for i in (1, 4, 0, 3, 5, 6, 8, 2, 7)))
    v = vc.reshape(*lead, 4, 4, 2, 2, d // 16, 2, 8)  # t kt n e dt r g
    v = v.permute(*range(a), *(a + i for i in (4, 6, 0, 1, 3, 5, 2)))
    k, v = ((x[..., 0] | (x[..., 1] << 4)).reshape(*lead, 32 * d) for x in (k, v))
    kp, vp = (x.reshape(*lead, 4, 4, 2, 2, g, 2).permute(*range(a), *(a + i for i in (0, 3, 1, 2, 4, 5))).contiguous()
              .view(torch.uint8).reshape(*lead, 256 * g) for x in (kp, vp))
    return torch.cat((k, kp, v, vp), -1)


def rotate(x, cos, sin, rotary, interleaved):
    if not rotary:
        return x
    a, b = (x[..., 0:rotary:2], x[..., 1:rotary:2]) if interleaved else (x[..., : rotary // 2], x[..., rotary // 2 : rotary])
    cos, sin = cos[:, None], sin[:, None]
    a, b = a * cos - b * sin, b * cos + a * sin
    r = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((r, x[..., rotary:]), -1)


def quantise(x):
    """Codes, f16 (scale, minimum) and the values they stand for, of [..., D] in 32 bits."""
    x = torch.nan_to_num(x, nan=0.0).clamp(-CLAMP, CLAMP).unflatten(-1, (-1, GROUP))
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    p = torch.cat(((high - low) / torch.full_like(low, 15.0), low), -1).half()
    scale, low = p[..., 0:1].float(), p[..., 1:2].float()
    c = torch.where(scale > 0, ((x - low) / scale).round().clamp(0, 15), 0.0)
    return c.to(torch.uint8).flatten(-2), p, (c * scale + low).flatten(-2)


def plain_append(s):
    case = s["case"]
    d, dtype = case["dim"], DTYPES[case["dtype"]]
    cos, sin = s["cos"][s["row_pos"]], s["sin"][s["row_pos"]]
    q = rotate(s["q"].float(), cos, sin, case["rotary"], case["interleaved"])
    k = rotate(s["k"].float(), cos, sin, case["rotary"], case["interleaved"])
    kc, kp, kx = quantise(k)
    vc, vp, vx = quantise(s["v"].float())
    # the touched pages with the new rows in their places
    seq, block = s["touched"][:, 0], s["touched"][:, 1]
    page = s["page_table"][seq, block].long()
    chunks = s["pages"][page]
    codes = [key_codes(chunks, d), value_codes(chunks, d)]
    scales = [params(chunks, d, at).half() for at in (32 * d, 64 * d + 256 * (d // GROUP))]
    at, slot = s["row_touched"], s["row_pos"] % PAGE
    for old, new in zip(codes + scales, (kc, vc, kp, vp)):
        old[at, :, slot] = new
    s["pages"][page] = pack(codes[0], scales[0], codes[1], scales[1], d)
    # bounds of the tokens that the pages hold
    x = values_of(codes[0], scales[0].float())
    held = (block[:, None] * PAGE + torch.arange(PAGE, device="cuda") < s["seq_len"][seq][:, None])[:, None, :, None]
    high = torch.where(held, x, -math.inf).amax(-2)
    low = torch.where(held, x, math.inf).amin(-2)
    top = torch.maximum(high.abs(), low.abs()).amax(-1)
    scale = top / torch.full_like(top, 127.0)
    div = scale[..., None]
    high = torch.where(div > 0, (high / div).ceil().clamp(-127, 127), 0.0)
    low = torch.where(div > 0, (low / div).floor().clamp(-127, 127), 0.0)
    s["bounds"][page] = torch.stack((high, low), -2).to(torch.int8)
    s["bound_scale"][page] = scale
    return q.to(dtype), kx.to(dtype), vx.to(dtype), s["bounds"], s["bound_scale"]


def plain_select(s):
    case = s["case"]
    kv, seqs, want = case["kv_heads"], case["seqs"], case["n_select"]
    group = case["heads"] // kv
    q = s["q"].float()
    top = q.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(top) & (top > 0)
    scale = torch.where(fine, top / torch.full_like(top, 127.0), 0.0)
    q8 = torch.where(fine, (q / scale).round().clamp(-127, 127), 0.0)
    q8 = torch.cat((q8.clamp(min=0), q8.clamp(max=0)), -1)
    # rows of each sequence, padded to the longest
    slot = torch.arange(s["n_rows"], device="cuda") - s["row_offset"][s["row_seq"]]
    rows = torch.zeros(seqs, s["max_rows"], kv, group, q8.shape[-1], device="cuda")
    rows[s["row_seq"], slot] = q8.unflatten(1, (kv, group))
    b = s["bounds"][s["page_table"].long()].float().flatten(-2)  # [seqs, blocks, kv, 2 D]
    dots = rows.permute(0, 2, 1, 3, 4).flatten(2, 3) @ b.permute(0, 2, 3, 1)
    dots = dots.unflatten(2, (s["max_rows"], group))[s["row_seq"], :, slot]  # [n, kv, group, blocks]
    score = (dots * scale.unflatten(1, (kv, group))).amax(2)
    score = score * s["bound_scale"][s["page_table"].long()].transpose(1, 2)[s["row_seq"]]
    at, last = torch.arange(score.shape[-1], device="cuda"), (s["row_pos"] // PAGE)[:, None, None]
    rank = torch.where((at < case["first"]) | (at > last - case["recent"]), math.inf, score)
    rank = torch.where(at <= last, rank, -math.inf)
    rank, ids = rank.sort(dim=-1, descending=True, stable=True)
    blocks = score.shape[-1]
    ids = torch.where(rank == -math.inf, blocks, ids)[..., :want].sort(-1).values
    got = torch.where(ids < blocks, score.gather(-1, ids.clamp(max=blocks - 1)), -math.inf)
    ids = torch.where(ids < blocks, ids, -1)
    pad = (0, want - ids.shape[-1])
    return (torch.nn.functional.pad(ids, pad, value=-1).int(), torch.nn.functional.pad(got, pad, value=-math.inf))


def plain_attend(s):
    case = s["case"]
    d, kv, seqs, dtype = case["dim"], case["kv_heads"], case["seqs"], DTYPES[case["dtype"]]
    group = case["heads"] // kv
    dev = s["q"].device
    q = s["q"].float().unflatten(1, (kv, group))
    if case["n_select"]:
        block = s["selected"].long()  # [n, kv, m]
        page = s["page_table"].long()[s["row_seq"][:, None, None], block.clamp(min=0)]
        k, v = keys_and_values(s["pages"][page, torch.arange(kv, device=dev)[:, None]], d)
        k, v = k.flatten(2, 3), v.flatten(2, 3)  # [n, kv, m 64, D]
        at = (block[..., None] * PAGE + torch.arange(PAGE, device=dev)).flatten(2)
        pos, length = s["row_pos"][:, None, None], s["seq_len"][s["row_seq"]][:, None, None]
        see = (at >= 0) & (at < length) & (at <= pos if case["causal"] else at < length)
        if case["window"]:
            see &= at > pos - case["window"]
        if case["bits"]:
            word = s["key_bits"][s["row_seq"][:, None, None], at.clamp(min=0) // 32]
            see &= ((word >> (at % 32)) & 1) > 0
        see = see[:, :, None]
    else:
        # rows of each sequence, padded to the longest
        slot = torch.arange(s["n_rows"], device=dev) - s["row_offset"][s["row_seq"]]
        rows = torch.zeros(seqs, s["max_rows"], kv, group, d, device=dev)
        rows[s["row_seq"], slot] = q
        pos = torch.zeros(seqs, s["max_rows"], dtype=torch.int64, device=dev)
        pos[s["row_seq"], slot] = s["row_pos"]
        q = rows.permute(0, 2, 1, 3, 4).flatten(2, 3)
        k, v = keys_and_values(s["pages"][s["page_table"].long()], d)  # [seqs, blocks, kv, 64, D]
        k, v = (x.transpose(1, 2).flatten(2, 3) for x in (k, v))
        at = torch.arange(k.shape[2], device=dev)
        pos = pos[:, :, None]
        see = (at < s["seq_len"][:, None, None]) & (at <= pos if case["causal"] else at + pos >= 0)
        if case["window"]:
            see &= at > pos - case["window"]
        if case["bits"]:
            see &= ((s["key_bits"][:, at // 32] >> (at % 32)) & 1)[:, None] > 0
        see = see[:, None].repeat_interleave(group, 2)
    # a value behind a mask takes no part, whatever it is
    score = torch.where(see, (q @ k.transpose(-1, -2)) * s["scale"], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = (score - top).exp()
    total = p.sum(-1, keepdim=True)
    out = torch.where(total > 0, (p @ v) / total, 0.0)
    lse = (top + total.log()).squeeze(-1)
    if not case["n_select"]:
        out = out.unflatten(2, (s["max_rows"], group))[s["row_seq"], :, slot]
        lse = lse.unflatten(2, (s["max_rows"], group))[s["row_seq"], :, slot]
    return out.flatten(1, 2).to(dtype), lse.flatten(1, 2).contiguous()


# ------------------------------------------------------------------ the same in 64 bits
def exact(case, seed):
    s = prepare(dict(case), seed)
    return {"append": exact_append, "select": exact_select, "attend": exact_attend}[case["op"]](case, s)


def place(token, dim, d):
    """Byte and nibble shift of (token, dimension) in the key codes and in the value codes, and the pair of its params."""
    groups = d // GROUP
    g1, kt, r, g0 = token // 16, token % 16 // 4, token % 4 // 2, token % 2
    t, j, n, e = dim % 64 // 16, dim % 16 // 4, dim % 4 // 2, dim % 2
    key = (((((kt * groups + dim // 64) * 8 + 2 * g1 + g0) * 4 + t) * 4 + j) * 2 + e) * 2 + r
    pair = ((2 * g1 + g0) * 4 + kt) * 2 + r
    t, kt, m, e = token // 16, token % 16 // 4, token % 4 // 2, token % 2
    value = ((((dim // 16 * 8 + dim % 8) * 4 + t) * 4 + kt) * 2 + e) * 2 + dim % 16 // 8
    return key, 4 * n, value, 4 * m, pair * groups + dim // 64


def decoded(chunks, d):
    """Keys and values [..., 64, D] in 64 bits, each element looked up by its place."""
    token, dim = torch.meshgrid(torch.arange(PAGE, device="cuda"), torch.arange(d, device="cuda"), indexing="ij")
    key, kshift, value, vshift, pair = place(token, dim, d)
    half = 32 * d + 256 * (d // GROUP)
    got = []
    for at, byte, shift in ((0, key, kshift), (half, value, vshift)):
        c = (chunks[..., at + byte] >> shift.to(torch.uint8)) & 15
        p = chunks[..., at + 32 * d : at + half].contiguous().view(torch.float16).double()
        got.append(c.double() * p[..., 2 * pair] + p[..., 2 * pair + 1])
    return got


def exact_append(case, s):
    d, rot, dtype = case["dim"], case["rotary"], DTYPES[case["dtype"]]
    i = torch.arange(rot // 2, device="cuda")
    first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + rot // 2)
    cos, sin = (x[s["row_pos"]].double()[:, None] for x in (s["cos"], s["sin"]))
    outs, held = [], {}
    for name in ("q", "k", "v"):
        x = s[name].double().clone()
        if name != "v" and rot:
            a, b = x[..., first].clone(), x[..., second].clone()
            x[..., first], x[..., second] = a * cos - b * sin, b * cos + a * sin
        if name != "q":
            y = x.reshape(*x.shape[:-1], -1, GROUP)
            low, high = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
            scale, low = ((high - low) / 15).half().double(), low.half().double()
            x = (((y - low) / scale).round().clamp(0, 15) * scale + low).reshape(x.shape)
            held[name] = x
        outs.append(x)
    scale = s["bound_scale"].double()
    for j, (seq, block) in enumerate(s["touched"].tolist()):
        page = int(s["page_table"][seq, block])
        count = min(PAGE, int(s["seq_len"][seq]) - block * PAGE)
        k = decoded(s["pages"][page], d)[0]
        mine = s["row_touched"] == j
        k[:, s["row_pos"][mine] % PAGE] = held["k"][mine].transpose(0, 1)
        scale[page] = k[:, :count].abs().amax((1, 2)) / 127
    return (*outs, None, scale)


def exact_select(case, s):
    kv, want = case["kv_heads"], case["n_select"]
    group = case["heads"] // kv
    q = s["q"].double()
    scale = q.abs().amax(-1, keepdim=True) / 127
    q8 = torch.where(scale > 0, (q / scale).round(), 0.0)
    got = torch.full((s["n_rows"], kv, want), -math.inf, dtype=torch.float64, device="cuda")
    offset, lens = s["row_offset"].tolist(), s["seq_len"].tolist()
    for i, length in enumerate(lens):
        lo, hi = offset[i], offset[i + 1]
        pages = s["page_table"][i, : -(-length // PAGE)].long()
        for head in range(kv):
            high, low = s["bounds"][pages, head].double().unbind(1)
            best = None
            for m in range(head * group, (head + 1) * group):
                x = q8[lo:hi, m]
                t = (x.clamp(min=0) @ high.T + x.clamp(max=0) @ low.T) * scale[lo:hi, m]
                best = t if best is None else torch.maximum(best, t)
            score = best * s["bound_scale"][pages, head].double()
            last = s["row_pos"][lo:hi, None] // PAGE
            at = torch.arange(len(pages), device="cuda")
            key = torch.where((at < case["first"]) | (at > last - case["recent"]), math.inf, score)
            key = torch.where(at <= last, key, -math.inf)
            order = key.sort(dim=-1, descending=True, stable=True).indices
            order = torch.where(key.gather(-1, order) == -math.inf, len(pages), order)[:, :want].sort(-1).values
            score = torch.nn.functional.pad(score, (0, 1), value=-math.inf)
            got[lo:hi, head, : order.shape[1]] = score.gather(-1, order)
    return None, got


def exact_attend(case, s):
    d, kv = case["dim"], case["kv_heads"]
    group = case["heads"] // kv
    out = torch.zeros(s["n_rows"], case["heads"], d, dtype=torch.float64, device="cuda")
    lse = torch.full((s["n_rows"], case["heads"]), -math.inf, dtype=torch.float64, device="cuda")
    offset, lens = s["row_offset"].tolist(), s["seq_len"].tolist()
    for i, length in enumerate(lens):
        lo, hi = offset[i], offset[i + 1]
        pages = s["page_table"][i, : -(-length // PAGE)].long()
        at, pos = torch.arange(length, device="cuda"), s["row_pos"][lo:hi, None]
        see = at <= pos if case["causal"] else torch.ones(hi - lo, length, dtype=torch.bool, device="cuda")
        if case["window"]:
            see = see & (at > pos - case["window"])
        if case["bits"]:
            see = see & ((s["key_bits"][i].long()[at // 32] >> (at % 32)) & 1).bool()
        for head in range(kv):
            k, v = (x.reshape(-1, d)[:length] for x in decoded(s["pages"][pages, head], d))
            mine = see
            if case["n_select"]:
                chosen = torch.zeros(hi - lo, len(pages) + 1, dtype=torch.bool, device="cuda")
                ids = s["selected"][lo:hi, head].long()
                chosen.scatter_(1, torch.where(ids < 0, len(pages), ids), True)
                mine = mine & chosen[:, at // PAGE]
            for m in range(head * group, (head + 1) * group):
                score = (s["q"][lo:hi, m].double() @ k.T) / math.sqrt(d)
                score = torch.where(mine, score, -math.inf)
                lse[lo:hi, m] = torch.logsumexp(score, -1)
                weight = torch.where(mine, (score - lse[lo:hi, m, None]).exp(), 0.0)
                out[lo:hi, m] = weight @ v
    return out, lse
