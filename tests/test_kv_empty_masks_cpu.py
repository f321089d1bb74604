"""A mask or a list of blocks that holds nothing has no address; it must not be taken for none at all."""
import pytest
import torch

from gofann import kv_cache as KV
from test_kv_devices_cpu import setting, there


class Library:
    """Notes the attention call's mask."""

    def __getattr__(self, name):
        def call(*args):
            if not name.endswith("bytes"):
                p = args[2]._obj
                self.seen = (p.key_bits, p.key_words, p.selected)
            return 256 if name.endswith("bytes") else 0
        return call


def test_no_words_hide_every_token(monkeypatch):
    cache, batch, calls = setting()
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    cache._lib = Library()
    bits = there(torch.zeros(1, 0, dtype=torch.int32))
    assert bits.data_ptr() == 0
    cache.attend(batch, calls["attend"]["q"], key_bits=bits)
    mask, words, _ = cache._lib.seen
    assert mask and words == 0
    cache.attend(batch, calls["attend"]["q"])
    assert cache._lib.seen == (None, 0, None)


def test_no_selected_blocks_are_refused():
    cache = KV.KVCache.empty(4, 2, 64, device="cpu")
    batch = KV.KVBatch(torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32),
                       torch.tensor([0, 1], dtype=torch.int32), 1, 1)
    with pytest.raises(ValueError, match="width from 1"):
        cache.attend(batch, torch.zeros(1, 2, 64, dtype=torch.bfloat16), selected=torch.zeros(1, 2, 0, dtype=torch.int32))
