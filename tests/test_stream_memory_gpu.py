"""The example that streams a tracker's memory through the quantised cache: projection, write over the oldest frame, attention
over the ring, read back."""
import importlib.util
import os

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("qtype,quantised", [(2, 0.5), (3, 0.5), (8, 0.04)])
@pytest.mark.parametrize("feat,frames,slots", [(6, 3, 7), (24, 9, 4)])
def test_stream_memory(s3b, qtype, quantised, feat, frames, slots):
    """On the values held, every rounding of the attention is to f16 (2^-11 a step, a handful of steps); on the unquantised
    ones half a code step a value, 1/16 of a block's range in 4 bits (keys and values: at most the sum of both)."""
    spec = importlib.util.spec_from_file_location("stream_memory", os.path.join(ROOT, "examples", "stream_memory.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    out, held, full, (cache, plain) = mod.run(feat, frames, slots, qtype, seed=feat)
    off = lambda x, y: ((x.double() - y).norm() / y.norm()).item()  # noqa: E731
    assert off(out, held) < 8 * 2.0 ** -11
    assert off(out, full) < quantised
    tokens = feat * feat + 4
    assert cache == s3b.kv_cache_bytes(qtype, 1, 256, 64, slots * -(-tokens // 64)) and plain == 1024 * slots * tokens
