"""The cache operators together: the decoding example at small sizes."""
import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


def example():
    spec = importlib.util.spec_from_file_location(
        "kv_decode", Path(__file__).resolve().parents[1] / "examples" / "kv_decode.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("head_dim", [64, 128])
def test_decoding_over_the_cache(head_dim):
    # 703 tokens, in chunks of 300: 11 blocks.  A value's step is 1/15 of a group of 64's range (about 4.8
    # deviations for normal numbers), which leaves an error of 0.32 / sqrt(12) = 0.092 deviations a value, uniform
    # and independent, in an output that averages as the values do; the keys' errors shift weight between tokens by
    # about as much.  Together about 0.13 of the output, taken twice.
    dense, picked, _ = example().run(700, 3, 11, seqs=2, chunk=300, heads=8, kv_heads=2, head_dim=head_dim, width=256)
    assert dense < 0.26
    # all blocks picked: the same tokens, so only the order of sums and 16-bit roundings differ
    assert abs(picked - dense) < 0.01


def test_fewer_blocks_read_less():
    dense, picked, _ = example().run(640, 1, 4, seqs=1, chunk=640, heads=4, kv_heads=4, head_dim=64, width=128)
    assert dense < 0.26 and picked > dense
