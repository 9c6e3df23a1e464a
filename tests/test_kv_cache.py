"""Host side of the quantised key / value cache: sizes and refusals that need no GPU."""
import pytest


@pytest.mark.parametrize("qtype", [2, 3, 8])
@pytest.mark.parametrize("heads,d,page,pages", [(1, 64, 16, 1), (5, 128, 48, 7), (8, 256, 5184, 3)])
def test_bytes_are_those_of_the_formats_rows(s3b, qtype, heads, d, page, pages):
    assert s3b.kv_cache_bytes(qtype, heads, d, page, pages) == 2 * s3b.row_size(qtype, d) * heads * page * pages


@pytest.mark.parametrize("qtype,heads,d,page,pages", [
    (1, 1, 64, 16, 1), (2, 0, 64, 16, 1), (2, -1, 64, 16, 1), (2, 1, 96, 16, 1), (2, 1, 32, 16, 1), (2, 1, 64, 0, 1),
    (2, 1, 64, 24, 1), (2, 1, 64, -16, 1), (2, 1, 64, 16, 0), (2, 1, 64, 16, -1), (8, 2 ** 30, 256, 2 ** 30, 1),
    (2, 2 ** 20, 64, 2 ** 20, 2 ** 62)])
def test_bytes_refuses(s3b, qtype, heads, d, page, pages):
    with pytest.raises(s3b.S3BError):
        s3b.kv_cache_bytes(qtype, heads, d, page, pages)


class _Tensor:
    """What the checks of the cache's calls look at of a tensor, on a GPU that this machine need not have."""

    def __init__(self, device, dtype, *shape):
        self.device_index, self.dtype, self.shape, self.is_cuda = device, dtype, shape, device >= 0

    def get_device(self):
        return self.device_index

    def dim(self):
        return len(self.shape)

    def numel(self):
        n = 1
        for x in self.shape:
            n *= x
        return n

    def element_size(self):
        return 1

    def is_contiguous(self):
        return True

    def stride(self, dim=None):
        s = [1]
        for x in self.shape[:0:-1]:
            s.insert(0, s[0] * x)
        return tuple(s) if dim is None else s[dim]

    def data_ptr(self):
        return 4096


class _Library:
    """Counts the calls that pass the checks."""

    def __init__(self):
        self.calls = 0

    def __getattr__(self, name):
        def call(*args):
            self.calls += 1
            return 0
        return call


@pytest.mark.parametrize("wrong", ["cache", "k", "v", "slots", "q", "out", "lse", "pages", "lengths", None])
def test_tensors_of_another_gpu_are_refused(s3b, wrong):
    torch = pytest.importorskip("torch")

    def at(name, dtype, *shape):
        return _Tensor(1 if name == wrong else 0, dtype, *shape)

    engine = s3b.Engine.__new__(s3b.Engine)
    engine._L, engine.device, engine.h = _Library(), 0, None
    cache = s3b.KVCache(2, 4, 16, 2, 64, data=at("cache", torch.uint8, s3b.kv_cache_bytes(2, 2, 64, 16, 4)))
    k, v = (at(n, torch.float32, 3, 2, 64) for n in "kv")
    slots = at("slots", torch.int64, 3)
    q, out = (at(n, torch.float16, 1, 5, 4, 64) for n in ("q", "out"))
    calls = [(("cache", "k", "v", "slots"), lambda: engine.cache_write(cache, k, v, slots)),
             (("cache", "k", "v", "slots"), lambda: engine.cache_read(cache, slots, k, v)),
             (("cache", "v", "slots"), lambda: engine.cache_read(cache, slots, None, v)),
             (("cache", "q", "out", "lse", "pages", "lengths"),
              lambda: engine.cache_attention(cache, q, out, at("pages", torch.int32, 1, 4), at("lengths", torch.int32, 1), 0.125,
                                             lse=at("lse", torch.float32, 1, 5, 4)))]
    for names, call in calls:
        before = engine._L.calls
        if wrong in names:
            with pytest.raises(s3b.S3BError):
                call()
            assert engine._L.calls == before
        else:
            call()
            assert engine._L.calls == before + 1
