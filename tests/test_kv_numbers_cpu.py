"""Numbers that the C structures' 32 bits do not hold are refused, not wrapped."""
import pytest
import torch

from gofann import kv_cache as KV
from test_kv_devices_cpu import setting


class Library:
    def __getattr__(self, name):
        return lambda *args: 256 if name.endswith("bytes") else 0


@pytest.fixture()
def ready(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    cache, batch, calls = setting()
    cache._lib = Library()
    return cache, batch, calls


@pytest.mark.parametrize("window", [-1, 1 << 32, (1 << 32) + 5])
def test_windows(ready, window):
    cache, batch, calls = ready
    with pytest.raises(ValueError, match="window"):
        cache.attend(batch, calls["attend"]["q"], window=window)
    cache.attend(batch, calls["attend"]["q"], window=(1 << 32) - 1)


@pytest.mark.parametrize("first,recent,n", [(-1, 1, 3), (1 << 32, 1, 3), (1, -(1 << 32), 3), (0, (1 << 32) + 1, 3)])
def test_kept_blocks(ready, first, recent, n):
    cache, batch, calls = ready
    with pytest.raises(ValueError, match="blocks of n_select"):
        cache.select(batch, calls["select"]["q"], n, first=first, recent=recent)
    cache.select(batch, calls["select"]["q"], 3, first=1, recent=2)
