"""Tensors on another device than the cache are refused before a kernel sees their addresses."""
import pytest
import torch

from gofann import kv_cache as KV

BF16 = torch.bfloat16


class OnGpu(torch.Tensor):
    """Host memory that says it is on GPU 0; nothing here gets as far as a kernel."""

    def get_device(self):
        return 0


def there(x):
    return x.as_subclass(OnGpu)


def setting():
    """A cache and a batch that seem to be on GPU 0, and the arguments of each call."""
    cache = KV.KVCache.empty(4, 2, 64, device="cpu")
    cache._index = 0
    batch = KV.KVBatch(there(torch.zeros(1, 4, dtype=torch.int32)), there(torch.ones(1, dtype=torch.int32)),
                       there(torch.tensor([0, 1], dtype=torch.int32)), 1, 1)
    x = lambda: there(torch.zeros(1, 2, 64, dtype=BF16))  # noqa: E731
    table = lambda: there(torch.zeros(9, 32))  # noqa: E731
    ints = lambda *n: there(torch.zeros(*n, dtype=torch.int32))  # noqa: E731
    calls = {
        "append": dict(q=x(), k=x(), v=x(), cos=table(), sin=table(), rotary_dim=64, positions=ints(1), q_out=x(), k_out=x(),
                       v_out=x()),
        "select": dict(q=x(), n_select=3, ids=ints(1, 2, 3), scores=there(torch.zeros(1, 2, 3))),
        "attend": dict(q=x(), selected=ints(1, 2, 3), key_bits=ints(1, 8), out=x(), lse=there(torch.zeros(1, 2))),
    }
    return cache, batch, calls


@pytest.mark.parametrize("op,name", [(op, name) for op, args in setting()[2].items() for name, x in args.items()
                                     if isinstance(x, torch.Tensor)])
def test_a_host_tensor_is_refused(op, name):
    cache, batch, calls = setting()
    args = dict(calls[op])
    args[name] = args[name].as_subclass(torch.Tensor)
    with pytest.raises(ValueError, match=rf"^{name} is on cpu, the cache on cuda:0"):
        getattr(cache, op)(batch, **args)


@pytest.mark.parametrize("op", ["append", "select", "attend"])
def test_a_batch_of_another_device_is_refused(op):
    cache, _, calls = setting()
    batch = KV.KVBatch(torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32),
                       torch.tensor([0, 1], dtype=torch.int32), 1, 1)
    with pytest.raises(ValueError, match="the batch is on cpu"):
        getattr(cache, op)(batch, **calls[op])


@pytest.mark.parametrize("op", ["append", "select", "attend"])
def test_a_cache_in_host_memory_is_refused(op):
    _, _, calls = setting()
    plain = lambda x: x.as_subclass(torch.Tensor) if isinstance(x, torch.Tensor) else x  # noqa: E731
    batch = KV.KVBatch(torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32),
                       torch.tensor([0, 1], dtype=torch.int32), 1, 1)
    with pytest.raises(ValueError, match="run on a GPU"):
        getattr(KV.KVCache.empty(4, 2, 64, device="cpu"), op)(batch, **{k: plain(v) for k, v in calls[op].items()})


def test_parts_of_a_cache_and_of_a_batch_are_on_one_device():
    pages = torch.zeros(4, 2, KV.chunk_bytes(64), dtype=torch.uint8)
    bounds, scale = torch.zeros(4, 2, 2, 64, dtype=torch.int8), torch.zeros(4, 2)
    for b, s in ((bounds.to("meta"), scale), (bounds, scale.to("meta"))):
        with pytest.raises(ValueError, match="pages on cpu"):
            KV.KVCache(64, pages=pages, bounds=b, bound_scale=s)
    args = (torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32),
            torch.tensor([0, 1], dtype=torch.int32), 1, 1)
    for status in (torch.zeros(1, dtype=torch.int32, device="meta"), torch.zeros(1), torch.zeros(0, dtype=torch.int32)):
        with pytest.raises(ValueError, match="status must be"):
            KV.KVBatch(*args, status=status)


@pytest.mark.parametrize("op", ["append", "select", "attend"])
def test_a_call_runs_on_the_device_of_its_cache(op, monkeypatch):
    """Another device is current: the library is called, and asked for its scratch, with the cache's device current, and
    the other one is current again behind the call."""
    cache, batch, calls = setting()
    current, seen = [3], []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.before

    class Library:
        def __getattr__(self, name):
            def call(*_):
                seen.append((name, current[0]))
                return 256 if name.endswith("bytes") else 0
            return call

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    cache._lib = Library()
    getattr(cache, op)(batch, **calls[op])
    assert seen and {device for _, device in seen} == {0}
    assert current == [3]
