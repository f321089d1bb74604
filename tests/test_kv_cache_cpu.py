"""The cache operators without a GPU: layouts, rotary tables and refusals."""
import ctypes as C
import math
import subprocess
from pathlib import Path

import pytest
import torch

import kv_reference as R
from gofann import _abi as A
from gofann import kv_cache as KV

ROOT = Path(__file__).resolve().parents[1]


def test_struct_layouts_match_c(tmp_path):
    names = {"gofann_kv_cache": A.KvCache, "gofann_kv_batch": A.KvBatch, "gofann_kv_append_params": A.KvAppendParams,
             "gofann_kv_select_params": A.KvSelectParams, "gofann_kv_attention_params": A.KvAttentionParams}
    lines = []
    for c, py in names.items():
        lines.append(f'printf("{c} %zu\\n", sizeof({c}));')
        lines += [f'printf("{c}.{f} %zu\\n", offsetof({c}, {f}));' for f, _ in py._fields_]
    src = tmp_path / "l.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "gofann.h"\nint main(void) {' + "\n".join(lines) +
                   'printf("page %u group %u select %u\\n", GOFANN_KV_PAGE, GOFANN_KV_GROUP, GOFANN_KV_MAX_SELECT); return 0; }')
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "l")], check=True)
    out = subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout.splitlines()
    assert out[-1] == f"page {A.KV_PAGE} group {A.KV_GROUP} select {A.KV_MAX_SELECT}"
    for line in out[:-1]:
        name, value = line.split()
        c, _, f = name.partition(".")
        assert int(value) == (getattr(names[c], f).offset if f else C.sizeof(names[c])), name


@pytest.mark.parametrize("d", [64, 128])
def test_chunk_layout_has_a_place_for_everything(d):
    assert KV.chunk_bytes(d) == R.chunk_size(d)
    nibbles, words = set(), set()
    for token in range(64):
        for dim in range(d):
            nibbles.add(R.key_place(token, dim, d))
            nibbles.add(R.value_place(token, dim, d))
        for grp in range(d // 64):
            words |= {R.param_place(token, grp, d, False), R.param_place(token, grp, d, True)}
    assert len(nibbles) == 2 * 64 * d and len(words) == 2 * d
    taken = {at for at, _ in nibbles} | {w + i for w in words for i in range(4)}
    assert taken == set(range(R.chunk_size(d)))


def test_unsupported_head_dim():
    assert A.lib().gofann_kv_chunk_bytes(96) == 0
    with pytest.raises(ValueError, match="head_dim 96"):
        KV.chunk_bytes(96)


@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "parts"])
def test_rope_tables(scaling):
    cos, sin = KV.rope_tables(40, 16, base=100.0, scaling=scaling, factor=4.0, original=30, device="cpu")
    m = 0.1 * math.log(4.0) + 1 if scaling == "parts" else 1.0
    base = 100.0 * 4.0 ** (16 / 14) if scaling == "ntk" else 100.0
    lo = max(math.floor(16 * math.log(30 / (2 * math.pi * 32)) / (2 * math.log(100.0))), 0)
    hi = min(math.ceil(16 * math.log(30 / (2 * math.pi * 1)) / (2 * math.log(100.0))), 7)
    for pos in (0, 1, 39):
        for i in range(8):
            f = base ** (-2 * i / 16)
            if scaling == "linear":
                f /= 4.0
            if scaling == "parts":
                r = min(max((i - lo) / max(hi - lo, 1e-3), 0.0), 1.0)
                f = f * (1 - r) + f / 4.0 * r
            assert abs(float(cos[pos, i]) - m * math.cos(pos * f)) < 1e-7 * 4
            assert abs(float(sin[pos, i]) - m * math.sin(pos * f)) < 1e-7 * 4
    # the fastest pair keeps its frequency under the scalings made for it
    if scaling in ("ntk", "parts"):
        assert abs(float(cos[1, 0]) - m * math.cos(1.0)) < 1e-6


def test_rope_tables_refuse():
    for kw in (dict(rotary_dim=3), dict(scaling="other"), dict(factor=0.5), dict(scaling="parts", factor=2.0)):
        with pytest.raises(ValueError):
            KV.rope_tables(4, **{"rotary_dim": 8, "device": "cpu", **kw})
    assert KV.rope_tables(4, 0, device="cpu")[0].shape == (4, 0)


# Addresses below are never followed: every refusal comes before any CUDA call.
def descriptors():
    cache = A.KvCache(pages=4096, bounds=4096, bound_scale=4096, n_pages=8, n_kv_heads=2, head_dim=64)
    batch = A.KvBatch(page_table=4096, seq_len=4096, row_offset=4096, n_seqs=2, max_pages=4, n_rows=2, max_rows=1)
    append = A.KvAppendParams(q=4096, k=4096, v=4096, q_stride=256, k_stride=128, v_stride=128, cos=4096, sin=4096,
                              q_out=8192, dtype=A.DTYPE_BF16, n_heads=4, n_positions=64, rotary_dim=64)
    select = A.KvSelectParams(q=4096, q_stride=256, ids=4096, scores=4096, dtype=A.DTYPE_F16, n_heads=4, n_select=4,
                              n_first=1, n_recent=1)
    attend = A.KvAttentionParams(q=4096, q_stride=256, out=8192, lse=4096, scale=0.1, dtype=A.DTYPE_BF16, n_heads=4, causal=1)
    return cache, batch, append, select, attend


def call(op, d, null=()):
    L = A.lib()
    cache, batch, append, select, attend = d
    c, b = (None if "cache" in null else C.byref(cache)), (None if "batch" in null else C.byref(batch))
    if op == "append":
        return L.gofann_kv_append(c, b, None if "params" in null else C.byref(append), None)
    p = None if "params" in null else C.byref(select if op == "select" else attend)
    fn = L.gofann_kv_select if op == "select" else L.gofann_kv_attention
    need = 0 if null else getattr(L, fn.__name__ + "_scratch_bytes")(c, b, p)
    return fn(c, b, p, None if "scratch" in null else 4096, need, None)


OPS = {"append": 2, "select": 3, "attend": 4}


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("null", ["cache", "batch", "params"])
def test_null_descriptors(op, null):
    assert call(op, descriptors(), (null,)) == A.ERR_INVALID
    assert b"null" in A.lib().gofann_last_error()


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("which,field,value,status", [
    ("cache", "head_dim", 96, A.ERR_UNSUPPORTED), ("cache", "n_kv_heads", 0, A.ERR_INVALID),
    ("cache", "n_kv_heads", 3, A.ERR_INVALID), ("cache", "n_pages", 0x80000000, A.ERR_UNSUPPORTED),
    ("batch", "max_pages", 0, A.ERR_INVALID), ("batch", "max_pages", (1 << 24) + 1, A.ERR_UNSUPPORTED),
    ("batch", "n_rows", (1 << 24) + 1, A.ERR_UNSUPPORTED), ("batch", "n_seqs", 0, A.ERR_INVALID),
    ("batch", "seq_len", None, A.ERR_INVALID), ("batch", "row_offset", None, A.ERR_INVALID),
    ("batch", "page_table", None, A.ERR_INVALID), ("params", "dtype", A.DTYPE_F32, A.ERR_INVALID),
    ("params", "n_heads", 0, A.ERR_INVALID), ("params", "n_heads", 3, A.ERR_INVALID),
    ("params", "n_heads", 65536, A.ERR_UNSUPPORTED), ("params", "q_stride", 255, A.ERR_INVALID),
    ("params", "q", 4097, A.ERR_INVALID)])
def test_shared_refusals(op, which, field, value, status):
    d = descriptors()
    setattr({"cache": d[0], "batch": d[1], "params": d[OPS[op]]}[which], field, value)
    assert call(op, d) == status
    assert A.lib().gofann_last_error().startswith({"append": b"kv_append", "select": b"kv_select", "attend": b"kv_attention"}[op])


@pytest.mark.parametrize("op,which,field,value,status", [
    ("append", "cache", "pages", None, A.ERR_INVALID), ("append", "cache", "pages", 4104, A.ERR_INVALID),
    ("append", "cache", "bounds", None, A.ERR_INVALID), ("append", "cache", "bounds", 4104, A.ERR_INVALID),
    ("append", "params", "k", None, A.ERR_INVALID), ("append", "params", "v", None, A.ERR_INVALID),
    ("append", "params", "q_out", None, A.ERR_INVALID), ("append", "params", "q", None, A.ERR_INVALID),
    ("append", "params", "q_out", 8196, A.ERR_INVALID), ("append", "params", "k_out", 8196, A.ERR_INVALID),
    ("append", "params", "rotary_dim", 63, A.ERR_INVALID), ("append", "params", "rotary_dim", 66, A.ERR_INVALID),
    ("append", "params", "cos", None, A.ERR_INVALID), ("append", "params", "n_positions", 0, A.ERR_INVALID),
    ("append", "params", "k_stride", 127, A.ERR_INVALID), ("append", "params", "v_stride", 127, A.ERR_INVALID),
    ("append", "params", "v", 4097, A.ERR_INVALID),
    ("select", "cache", "bounds", None, A.ERR_INVALID), ("select", "cache", "bound_scale", None, A.ERR_INVALID),
    ("select", "cache", "bounds", 4104, A.ERR_INVALID), ("select", "params", "q", None, A.ERR_INVALID),
    ("select", "params", "ids", None, A.ERR_INVALID), ("select", "params", "n_select", 0, A.ERR_UNSUPPORTED),
    ("select", "params", "n_select", 1025, A.ERR_UNSUPPORTED), ("select", "params", "n_recent", 4, A.ERR_INVALID),
    ("select", "params", "n_first", 5, A.ERR_INVALID), ("select", "params", "n_recent", 0xFFFFFFFF, A.ERR_INVALID),
    ("attend", "cache", "pages", None, A.ERR_INVALID), ("attend", "cache", "pages", 4104, A.ERR_INVALID),
    ("attend", "params", "q", None, A.ERR_INVALID), ("attend", "params", "out", None, A.ERR_INVALID),
    ("attend", "params", "out", 8196, A.ERR_INVALID), ("attend", "params", "scale", float("nan"), A.ERR_INVALID),
    ("attend", "params", "scale", float("inf"), A.ERR_INVALID), ("attend", "params", "selected", 4096, A.ERR_INVALID)])
def test_own_refusals(op, which, field, value, status):
    d = descriptors()
    setattr({"cache": d[0], "batch": d[1], "params": d[OPS[op]]}[which], field, value)
    assert call(op, d) == status


def test_append_in_place_needs_contiguous_rows():
    d = descriptors()
    d[2].q_out, d[2].q_stride = d[2].q, 320
    assert call("append", d) == A.ERR_INVALID


@pytest.mark.parametrize("op", ["select", "attend"])
def test_scratch_is_checked(op):
    L = A.lib()
    d = descriptors()
    fn = L.gofann_kv_select if op == "select" else L.gofann_kv_attention
    p = C.byref(d[OPS[op]])
    need = getattr(L, fn.__name__ + "_scratch_bytes")(C.byref(d[0]), C.byref(d[1]), p)
    assert fn(C.byref(d[0]), C.byref(d[1]), p, None, need, None) == A.ERR_INVALID
    assert fn(C.byref(d[0]), C.byref(d[1]), p, 4100, need, None) == A.ERR_INVALID
    assert fn(C.byref(d[0]), C.byref(d[1]), p, 4096, need - 1, None) == A.ERR_CAPACITY


@pytest.mark.parametrize("op", OPS)
def test_no_rows_is_no_work(op):
    d = descriptors()
    d[1].n_rows = d[1].max_rows = 0
    assert call(op, d) == A.OK


def tensors():
    cache = KV.KVCache.empty(4, 2, 64, device="cpu")
    batch = KV.KVBatch(torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32),
                       torch.tensor([0, 1], dtype=torch.int32), 1, 1)
    return cache, batch


def test_python_refusals():
    cache, batch = tensors()
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="a cache needs"):
        KV.KVCache(64)
    with pytest.raises(ValueError, match="pages must be"):
        KV.KVCache(128, pages=cache.pages)
    with pytest.raises(ValueError, match="go together"):
        KV.KVCache(64, bounds=cache.bounds)
    with pytest.raises(ValueError, match="bounds must be"):
        KV.KVCache(64, bounds=cache.bounds.float(), bound_scale=cache.bound_scale)
    for args in ((batch.page_table.long(), batch.seq_len, batch.row_offset, 1, 1),
                 (batch.page_table, batch.seq_len, batch.seq_len, 1, 1),
                 (batch.page_table, batch.seq_len, batch.row_offset, 1, 2)):
        with pytest.raises(ValueError):
            KV.KVBatch(*args)
    with pytest.raises(TypeError):
        cache.attend(batch, x.float())
    with pytest.raises(ValueError, match="multiple"):
        cache.attend(batch, x[:, :1])
    with pytest.raises(ValueError, match="contiguous"):
        cache.attend(batch, torch.zeros(1, 64, 2, dtype=torch.bfloat16).transpose(1, 2))
    with pytest.raises(ValueError, match="rows"):
        cache.attend(batch, torch.zeros(2, 2, 64, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="selected"):
        cache.attend(batch, x, selected=torch.zeros(1, 2, 4))
    with pytest.raises(ValueError, match="key_bits"):
        cache.attend(batch, x, key_bits=torch.zeros(2, 4, dtype=torch.int32))
    with pytest.raises(ValueError, match="out must be"):
        cache.attend(batch, x, out=torch.zeros(1, 2, 64))
    with pytest.raises(ValueError, match="ids must be"):
        cache.select(batch, x, 4, ids=torch.zeros(1, 2, 5, dtype=torch.int32))
    with pytest.raises(TypeError):
        cache.append(batch, None, x.float(), x.float())
    with pytest.raises(TypeError):
        cache.append(batch, x.half(), x, x)
    with pytest.raises(ValueError, match="cos and sin"):
        cache.append(batch, x, x, x, rotary_dim=64)
    with pytest.raises(ValueError, match="positions"):
        cache.append(batch, x, x, x, positions=torch.zeros(2, dtype=torch.int32))
