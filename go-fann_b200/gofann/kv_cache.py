"""A language model's key/value cache in 4 bits, searched like an index.

The cache operators of the C ABI (gofann_kv_append, gofann_kv_select,
gofann_kv_attention) on torch-managed device memory: new rows are rotated and
written in 4 bits, an int8 bound picks the blocks that a query reads, and
attention reads all blocks or the picked ones.

    cache = KVCache.empty(n_pages, n_kv_heads, head_dim)
    cos, sin = rope_tables(max_positions, rotary_dim)
    batch = KVBatch(page_table, seq_len, row_offset, n_rows, max_rows)
    q, _, _ = cache.append(batch, q, k, v, cos=cos, sin=sin, rotary_dim=rotary_dim)
    ids, _ = cache.select(batch, q, n_select=64, first=1, recent=2)
    out, lse = cache.attend(batch, q, selected=ids)

Calls run on the current stream of the cache's device, or on `stream`: then
their outputs and scratch are memory of that stream, and their arguments are
kept for it; the caller orders it behind what makes the arguments.  Scratch
belongs to the batch object, one for each stream, and is kept until the batch
object goes, as a captured graph needs it; graphs captured from one batch
object share it and are replayed one after the other.  Outputs carry no
gradient.  There is no CPU or torch fallback.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _abi as A

PAGE, GROUP = A.KV_PAGE, A.KV_GROUP
DTYPES = {torch.bfloat16: A.DTYPE_BF16, torch.float16: A.DTYPE_F16}


def chunk_bytes(head_dim: int) -> int:
    """Bytes of one (page, key/value head)."""
    n = int(A.lib().gofann_kv_chunk_bytes(head_dim))
    if n == 0:
        raise ValueError(f"head_dim {head_dim} is not supported (64 or 128)")
    return n


def rope_tables(n_positions: int, rotary_dim: int, base: float = 10000.0, scaling: str = "none",
                factor: float = 1.0, original: int = 0, beta_fast: float = 32.0, beta_slow: float = 1.0,
                magnitude: float | None = None, device="cuda"):
    """cos and sin tables [n_positions][rotary_dim / 2] (f32, computed in f64).

    scaling "none"; "linear": positions divided by `factor`; "ntk": the base
    raised to base * factor^(r / (r - 2)), which leaves the fastest pair alone
    and slows the slowest by `factor`; "parts": pairs that turn more than
    `beta_fast` times over the `original` context keep their frequency, those
    below `beta_slow` turns are divided by `factor`, with a linear ramp in the
    pair index between.  `magnitude` multiplies both tables (default 1, for
    "parts" 0.1 ln(factor) + 1)."""
    if rotary_dim < 0 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even")
    if scaling not in ("none", "linear", "ntk", "parts"):
        raise ValueError(f"unknown scaling {scaling!r}")
    if not factor >= 1.0:
        raise ValueError("factor must be at least 1")
    if scaling == "ntk" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    freq = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / max(rotary_dim, 1))
    if scaling == "linear":
        freq = freq / factor
    if scaling == "parts":
        if original <= 0:
            raise ValueError('"parts" needs the original context length')

        def pair(turns: float) -> float:  # the pair that turns this often over the original context
            return rotary_dim * math.log(original / (2 * math.pi * turns)) / (2 * math.log(base))

        lo = max(math.floor(pair(beta_fast)), 0)
        hi = math.ceil(pair(beta_slow))  # past the last pair where all turn more often
        ramp = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        freq = freq * (1 - ramp) + freq / factor * ramp
        if magnitude is None:
            magnitude = 0.1 * math.log(factor) + 1.0
    m = 1.0 if magnitude is None else magnitude
    angle = torch.arange(n_positions, dtype=torch.float64, device=device)[:, None] * freq.to(device)
    return (angle.cos() * m).float(), (angle.sin() * m).float()


def _elsewhere(x: torch.Tensor, index: int, name: str) -> ValueError:
    """A tensor that is not on the cache's device: a kernel would follow its address all the same."""
    return ValueError(f"{name} is on {x.device}, the cache on {f'cuda:{index}' if index >= 0 else 'cpu'}")


def _rows(x: torch.Tensor, rows: int, heads: int, dim: int, dtype, name: str, index: int) -> tuple[int, int]:
    """Address and row stride of [rows][heads][dim] with contiguous heads."""
    if x.shape != (rows, heads, dim):
        raise ValueError(f"{name} must be [{rows} rows][{heads}][{dim}], got {tuple(x.shape)}")
    if x.dtype is not dtype:
        raise TypeError(f"{name} is {x.dtype}, not {dtype}")
    stride = x.stride()
    if stride[2] != 1 or (heads > 1 and stride[1] != dim):
        raise ValueError(f"{name}: the heads of a row must be contiguous")
    if x.get_device() != index:
        raise _elsewhere(x, index, name)
    return x.data_ptr(), stride[0] if rows > 1 else heads * dim


def _out(x: torch.Tensor | None, shape: tuple, dtype, like: torch.Tensor, name: str, index: int) -> torch.Tensor:
    if x is None:
        return torch.empty(shape, dtype=dtype, device=like.device)
    if x.shape != shape or x.dtype is not dtype or not x.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {shape}")
    if x.get_device() != index:
        raise _elsewhere(x, index, name)
    return x


class KVBatch:
    """The sequences of a call and their query rows (gofann_kv_batch).

    page_table int32 [n_seqs][max_pages], seq_len int32 [n_seqs] (tokens in
    the cache, this call's rows among them), row_offset int32 [n_seqs + 1].
    The tensors stay on the device and may be updated in place between calls;
    n_rows = row_offset[-1] and max_rows, the longest sequence's rows, are the
    host's."""

    def __init__(self, page_table: torch.Tensor, seq_len: torch.Tensor, row_offset: torch.Tensor, n_rows: int,
                 max_rows: int, status: torch.Tensor | None = None):
        for name, t in (("page_table", page_table), ("seq_len", seq_len), ("row_offset", row_offset)):
            if t.dtype != torch.int32 or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous int32 tensor")
            if t.device != page_table.device:
                raise ValueError(f"{name} is on {t.device}, page_table on {page_table.device}")
        n_seqs = seq_len.numel()
        if seq_len.dim() != 1 or page_table.dim() != 2 or page_table.shape[0] != n_seqs or tuple(row_offset.shape) != (n_seqs + 1,):
            raise ValueError("page_table [n_seqs][max_pages], seq_len [n_seqs] and row_offset [n_seqs + 1] disagree")
        if n_rows < 0 or not 0 <= max_rows <= n_rows:
            raise ValueError(f"n_rows {n_rows} and max_rows {max_rows}")
        self.page_table, self.seq_len, self.row_offset = page_table, seq_len, row_offset
        self.n_seqs, self.n_rows, self.max_rows = n_seqs, int(n_rows), int(max_rows)
        if status is not None and (status.dtype != torch.int32 or status.numel() < 1 or status.device != page_table.device):
            raise ValueError(f"status must be an int32 tensor on {page_table.device}")
        self.status = status if status is not None else torch.zeros(1, dtype=torch.int32, device=page_table.device)
        self._index = page_table.get_device()
        self.struct = A.KvBatch(page_table=page_table.data_ptr(), seq_len=seq_len.data_ptr(),
                                row_offset=row_offset.data_ptr(), status=self.status.data_ptr(), n_seqs=n_seqs,
                                max_pages=int(page_table.shape[1]), n_rows=self.n_rows, max_rows=self.max_rows)
        self._ref = C.byref(self.struct)
        self._scratch = {}  # by stream: (address, bytes) of its newest buffer
        self._buffers = []  # all of them: a graph may hold an outgrown one's address
        self._needs = {}

    def scratch(self, stream: int, key: tuple, need) -> tuple[int, int]:
        """Address and size of the device scratch of a call on `stream`, the
        current one (kept, grown on demand); `need` tells the bytes, once for
        each `key`, a call's sizes."""
        n_bytes = self._needs.get(key)
        if n_bytes is None:
            n_bytes = self._needs[key] = max(int(need()), 256)
        got = self._scratch.get(stream)
        if got is None or got[1] < n_bytes:
            self._buffers.append(torch.empty(n_bytes, dtype=torch.uint8, device=self.page_table.device))
            got = self._scratch[stream] = (self._buffers[-1].data_ptr(), n_bytes)
        return got

    def check(self) -> None:
        """Raises where a call found a page, position, length or row out of range (synchronises)."""
        if int(self.status.item()) != A.OK:
            status = int(self.status.item())
            self.status.zero_()
            raise A.GofannError(status, "kv cache call (device)")


class KVCache:
    """Pages of a 4-bit key/value cache and the int8 bounds of their blocks."""

    def __init__(self, head_dim: int, pages: torch.Tensor | None = None, bounds: torch.Tensor | None = None,
                 bound_scale: torch.Tensor | None = None):
        size = chunk_bytes(head_dim)
        first = pages if pages is not None else bounds
        if first is None:
            raise ValueError("a cache needs pages or bounds")
        n_pages, n_kv = int(first.shape[0]), int(first.shape[1])
        if pages is not None and (tuple(pages.shape) != (n_pages, n_kv, size) or pages.dtype != torch.uint8 or
                                  not pages.is_contiguous()):
            raise ValueError(f"pages must be contiguous uint8 [n_pages][n_kv_heads][{size}]")
        if (bounds is None) != (bound_scale is None):
            raise ValueError("bounds and bound_scale go together")
        if bounds is not None and (tuple(bounds.shape) != (n_pages, n_kv, 2, head_dim) or bounds.dtype != torch.int8 or
                                   tuple(bound_scale.shape) != (n_pages, n_kv) or bound_scale.dtype != torch.float32 or
                                   not bounds.is_contiguous() or not bound_scale.is_contiguous()):
            raise ValueError(f"bounds must be contiguous int8 [n_pages][n_kv_heads][2][{head_dim}] and bound_scale "
                             "float32 [n_pages][n_kv_heads]")
        for t in (bounds, bound_scale):
            if t is not None and t.device != first.device:
                raise ValueError(f"bounds and bound_scale are on {t.device}, pages on {first.device}")
        self.head_dim, self.n_kv_heads, self.n_pages = head_dim, n_kv, n_pages
        self.pages, self.bounds, self.bound_scale = pages, bounds, bound_scale
        self.device = first.device
        self._index = first.get_device()
        self._lib = A.lib()
        self.struct = A.KvCache(pages=A.ptr(pages), bounds=A.ptr(bounds), bound_scale=A.ptr(bound_scale),
                                n_pages=n_pages, n_kv_heads=n_kv, head_dim=head_dim)
        self._ref = C.byref(self.struct)

    @classmethod
    def empty(cls, n_pages: int, n_kv_heads: int, head_dim: int, device="cuda") -> "KVCache":
        """An empty cache (pages hold nothing until rows are appended)."""
        return cls(head_dim,
                   pages=torch.zeros((n_pages, n_kv_heads, chunk_bytes(head_dim)), dtype=torch.uint8, device=device),
                   bounds=torch.zeros((n_pages, n_kv_heads, 2, head_dim), dtype=torch.int8, device=device),
                   bound_scale=torch.zeros((n_pages, n_kv_heads), dtype=torch.float32, device=device))

    def _away(self, stream):
        """What makes `stream` and the cache's device the current ones, or None where nothing has to: launches, outputs,
        scratch and the number of SMs that a call counts on are the current ones'."""
        if self._index < 0:
            return None
        if stream is not None:
            if stream.device_index != self._index:
                raise ValueError(f"the stream is of cuda:{stream.device_index}, the cache on cuda:{self._index}")
            return torch.cuda.stream(stream)
        try:
            return None if torch._C._cuda_getDevice() == self._index else torch.cuda.device(self._index)
        except RuntimeError:  # no driver: what is wrong with the arguments is said first
            return None

    def _keep(self, stream, batch: KVBatch, *tensors) -> None:
        """Keeps the memory of a call's arguments until `stream` has run it."""
        for t in (self.pages, self.bounds, self.bound_scale, batch.page_table, batch.seq_len, batch.row_offset, batch.status,
                  *tensors):
            if t is not None:
                t.record_stream(stream)

    def _on(self, batch: KVBatch) -> int:
        """The current stream; refuses what a kernel must not follow: a batch of another device, a cache in host memory."""
        if batch._index != self._index:
            raise ValueError(f"the batch is on {batch.page_table.device}, the cache on {self.device}")
        if self._index < 0:
            raise ValueError(f"the cache is on {self.device}: its operators run on a GPU")
        return torch._C._cuda_getCurrentRawStream(self._index)

    def _heads(self, q: torch.Tensor) -> int:
        shape = q.shape
        if len(shape) != 3 or shape[1] % self.n_kv_heads or not shape[1]:
            raise ValueError(f"queries must be [rows][heads][{self.head_dim}] with heads a multiple of {self.n_kv_heads}")
        if q.dtype not in DTYPES:
            raise TypeError(f"queries are {q.dtype}, not bfloat16 or float16")
        return shape[1]

    def append(self, batch: KVBatch, q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, cos=None, sin=None,
               rotary_dim: int = 0, interleaved: bool = False, positions=None, q_out=None, k_out=None, v_out=None,
               held: bool = False, stream=None):
        """Rotates q and k, writes k and v to the pages, renews the touched bounds.

        Returns the rotated queries and, where k_out / v_out are given or
        `held` is set, the keys and values as the cache holds them (else None)."""
        away = self._away(stream)
        if away is not None:
            with away:
                got = self.append(batch, q, k, v, cos, sin, rotary_dim, interleaved, positions, q_out, k_out, v_out, held)
            if stream is not None:
                self._keep(stream, batch, q, k, v, cos, sin, positions, q_out, k_out, v_out)
            return got
        d, n_kv, n, index = self.head_dim, self.n_kv_heads, batch.n_rows, self._index
        dtype = k.dtype
        if dtype not in DTYPES:
            raise TypeError(f"keys are {dtype}, not bfloat16 or float16")
        k_at, k_stride = _rows(k, n, n_kv, d, dtype, "k", index)
        v_at, v_stride = _rows(v, n, n_kv, d, dtype, "v", index)
        heads, q_at, q_stride, q_to, k_to, v_to = n_kv, None, 0, None, None, None
        if q is not None:
            heads = self._heads(q)
            q_at, q_stride = _rows(q, n, heads, d, dtype, "q", index)
            q_out = _out(q_out, (n, heads, d), dtype, k, "q_out", index)
            q_to = q_out.data_ptr()
        if held or k_out is not None:
            k_out = _out(k_out, (n, n_kv, d), dtype, k, "k_out", index)
            k_to = k_out.data_ptr()
        if held or v_out is not None:
            v_out = _out(v_out, (n, n_kv, d), dtype, k, "v_out", index)
            v_to = v_out.data_ptr()
        cos_at, sin_at, n_positions, positions_at = None, None, 0, None
        if rotary_dim:
            if cos is None or sin is None or cos.dtype is not torch.float32 or sin.dtype is not torch.float32 or \
                    cos.shape != sin.shape or cos.dim() != 2 or cos.shape[1] != rotary_dim // 2 or \
                    not cos.is_contiguous() or not sin.is_contiguous():
                raise ValueError(f"cos and sin must be contiguous float32 [positions][{rotary_dim // 2}]")
            if cos.get_device() != index:
                raise _elsewhere(cos, index, "cos")
            if sin.get_device() != index:
                raise _elsewhere(sin, index, "sin")
            cos_at, sin_at, n_positions = cos.data_ptr(), sin.data_ptr(), cos.shape[0]
        if positions is not None:
            if positions.dtype is not torch.int32 or positions.shape != (n,) or not positions.is_contiguous():
                raise ValueError("positions must be contiguous int32 [n_rows]")
            if positions.get_device() != index:
                raise _elsewhere(positions, index, "positions")
            positions_at = positions.data_ptr()
        now = self._on(batch)
        p = A.KvAppendParams(q_at, k_at, v_at, q_stride, k_stride, v_stride, cos_at, sin_at, positions_at, q_to, k_to,
                             v_to, DTYPES[dtype], heads, n_positions, rotary_dim, 1 if interleaved else 0)
        status = self._lib.gofann_kv_append(self._ref, batch._ref, C.byref(p), now)
        if status:
            A.check(status, "gofann_kv_append")
        return q_out if q is not None else None, k_out, v_out

    def select(self, batch: KVBatch, q: torch.Tensor, n_select: int, first: int = 1, recent: int = 1, ids=None,
               scores=None, stream=None):
        """Blocks that each row and key/value head reads: ids int32 and scores
        f32 [n_rows][n_kv_heads][n_select], ascending blocks, -1 / -inf fill."""
        away = self._away(stream)
        if away is not None:
            with away:
                got = self.select(batch, q, n_select, first, recent, ids, scores)
            if stream is not None:
                self._keep(stream, batch, q, ids, scores)
            return got
        heads, n, index = self._heads(q), batch.n_rows, self._index
        at, stride = _rows(q, n, heads, self.head_dim, q.dtype, "q", index)
        if not (0 <= first <= A.U32MAX and 0 <= recent <= A.U32MAX):
            raise ValueError(f"first {first} and recent {recent} (blocks of n_select {n_select})")
        shape = (n, self.n_kv_heads, n_select)
        ids = _out(ids, shape, torch.int32, q, "ids", index)
        scores = _out(scores, shape, torch.float32, q, "scores", index)
        now = self._on(batch)
        ref = C.byref(A.KvSelectParams(at, stride, ids.data_ptr(), scores.data_ptr(), DTYPES[q.dtype], heads, n_select,
                                       first, recent))
        scratch, size = batch.scratch(now, (0, heads, self.n_kv_heads, self.head_dim, n_select),
                                      lambda: self._lib.gofann_kv_select_scratch_bytes(self._ref, batch._ref, ref))
        status = self._lib.gofann_kv_select(self._ref, batch._ref, ref, scratch, size, now)
        if status:
            A.check(status, "gofann_kv_select")
        return ids, scores

    def attend(self, batch: KVBatch, q: torch.Tensor, scale: float | None = None, causal: bool = True, window: int = 0,
               selected=None, key_bits=None, out=None, lse=None, stream=None):
        """softmax(scale q.K^T) V over the cache: out like q, lse f32 [n_rows][heads].

        selected int32 [n_rows][n_kv_heads][width]: the blocks that each row
        reads (select's ids); key_bits int32 [n_seqs][words]: a bit per token,
        0 hides it (filtered out or evicted).  scale defaults to
        head_dim^-0.5."""
        away = self._away(stream)
        if away is not None:
            with away:
                got = self.attend(batch, q, scale, causal, window, selected, key_bits, out, lse)
            if stream is not None:
                self._keep(stream, batch, q, selected, key_bits, out, lse)
            return got
        heads, n, d, index = self._heads(q), batch.n_rows, self.head_dim, self._index
        at, stride = _rows(q, n, heads, d, q.dtype, "q", index)
        out = _out(out, (n, heads, d), q.dtype, q, "out", index)
        lse = _out(lse, (n, heads), torch.float32, q, "lse", index)
        if not 0 <= window <= A.U32MAX:
            raise ValueError(f"window {window} (0 for none, at most {A.U32MAX})")
        selected_at, n_select, bits_at, words = None, 0, None, 0
        if selected is not None:
            if selected.dtype is not torch.int32 or selected.dim() != 3 or not selected.is_contiguous() or \
                    selected.shape[:2] != (n, self.n_kv_heads) or not selected.shape[2]:
                raise ValueError(f"selected must be contiguous int32 [{n}][{self.n_kv_heads}][width from 1]")
            if selected.get_device() != index:
                raise _elsewhere(selected, index, "selected")
            selected_at, n_select = selected.data_ptr(), selected.shape[2]
        if key_bits is not None:
            if key_bits.dtype is not torch.int32 or key_bits.dim() != 2 or not key_bits.is_contiguous() or \
                    key_bits.shape[0] != batch.n_seqs:
                raise ValueError("key_bits must be contiguous int32 [n_seqs][words]")
            if key_bits.get_device() != index:
                raise _elsewhere(key_bits, index, "key_bits")
            # (no words hide every token; their tensor has no address, which would stand for no mask)
            bits_at, words = key_bits.data_ptr() or batch.page_table.data_ptr(), key_bits.shape[1]
        now = self._on(batch)
        ref = C.byref(A.KvAttentionParams(at, stride, selected_at, bits_at, out.data_ptr(), lse.data_ptr(),
                                          d ** -0.5 if scale is None else scale, DTYPES[q.dtype], heads, n_select, words,
                                          1 if causal else 0, window))
        scratch, size = batch.scratch(now, (1, heads, self.n_kv_heads, d, n_select),
                                      lambda: self._lib.gofann_kv_attention_scratch_bytes(self._ref, batch._ref, ref))
        status = self._lib.gofann_kv_attention(self._ref, batch._ref, ref, scratch, size, now)
        if status:
            A.check(status, "gofann_kv_attention")
        return out, lse
