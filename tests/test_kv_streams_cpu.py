"""Memory of calls on a stream of their own, without a GPU: where it is taken and how long it is kept."""
import pytest
import torch

from gofann import kv_cache as KV
from test_kv_devices_cpu import setting


class Stream:
    def __init__(self, handle, device_index=0):
        self.cuda_stream, self.device_index = handle, device_index


class World:
    """The current stream, a library that notes the stream it is given, tensors that note the streams they are kept for."""

    def __init__(self, monkeypatch, need):
        self.now, self.taken, self.given, self.kept = [11], [], [], {}
        world, empty = self, torch.empty

        class Context:
            def __init__(self, stream):
                self.stream = stream

            def __enter__(self):
                self.before, world.now[0] = world.now[0], self.stream.cuda_stream

            def __exit__(self, *_):
                world.now[0] = self.before

        class Library:
            def __getattr__(self, name):
                def call(*args):
                    if name.endswith("bytes"):
                        return need[0]
                    world.given.append(args[-1])
                    return 0
                return call

        def noted(*args, **kw):
            x = empty(*args, **kw)
            self.taken.append((self.now[0], x.data_ptr(), x.numel() * x.element_size()))
            return x

        monkeypatch.setattr(torch.cuda, "stream", Context)
        monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
        monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: self.now[0], raising=False)
        monkeypatch.setattr(torch, "empty", noted)
        monkeypatch.setattr(torch.Tensor, "record_stream",
                            lambda x, stream: self.kept.setdefault(x.data_ptr(), set()).add(stream.cuda_stream))
        self.library = Library()


def bare(args):
    """Without the outputs: the call makes them."""
    return {k: v for k, v in args.items() if k not in ("q_out", "k_out", "v_out", "ids", "scores", "out", "lse")}


@pytest.mark.parametrize("op", ["append", "select", "attend"])
def test_a_call_on_a_stream_takes_its_memory_there(op, monkeypatch):
    cache, batch, calls = setting()
    world = World(monkeypatch, [512])
    cache._lib = world.library
    args = bare(calls[op])
    getattr(cache, op)(batch, **args, stream=Stream(77))
    assert world.given == [77]
    assert world.taken and {stream for stream, *_ in world.taken} == {77}
    assert world.now == [11]
    for x in (*args.values(), cache.pages, cache.bounds, cache.bound_scale, batch.page_table, batch.seq_len, batch.row_offset,
              batch.status):
        if isinstance(x, torch.Tensor):
            assert world.kept[x.data_ptr()] == {77}


def test_a_stream_of_another_device_is_refused(monkeypatch):
    cache, batch, calls = setting()
    World(monkeypatch, [512])
    with pytest.raises(ValueError, match="the stream is of cuda:1, the cache on cuda:0"):
        cache.attend(batch, **calls["attend"], stream=Stream(77, 1))


def test_scratch_is_of_its_stream_and_is_kept(monkeypatch):
    """An outgrown buffer may be in a captured graph, or in use by a call in flight: it stays as long as the batch."""
    cache, batch, calls = setting()
    need = [512]
    world = World(monkeypatch, need)
    cache._lib = world.library
    cache.attend(batch, **calls["attend"])
    need[0] = 4096
    cache.select(batch, **calls["select"])   # grows it
    cache.attend(batch, **calls["attend"])
    assert [size for _, _, size in world.taken] == [512, 4096]
    cache.select(batch, **calls["select"], stream=Stream(77))
    cache.select(batch, **calls["select"], stream=Stream(77))
    assert [(stream, size) for stream, _, size in world.taken] == [(11, 512), (11, 4096), (77, 4096)]
    # nothing was freed: the addresses differ and the batch has all three
    assert len({at for _, at, _ in world.taken}) == 3
    assert [b.data_ptr() for b in batch._buffers] == [at for _, at, _ in world.taken]
