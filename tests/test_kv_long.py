"""Long caches, host side: tensors that the calls refuse before any kernel, on machines without a GPU too."""
import pytest

torch = pytest.importorskip("torch")
from test_kv_cache import _Library, _Tensor  # noqa: E402

KV, D, PAGE, PAGES, KEEP = 2, 64, 16, 4, 3


class _Strided(_Tensor):
    """As a tensor of which a test may change the strides."""

    def __init__(self, *args, strides=None):
        super().__init__(*args)
        self.strides = strides
        self.device = type("Device", (), {"type": "cuda"})()

    def stride(self, dim=None):
        s = self.strides or super().stride()
        return tuple(s) if dim is None else s[dim]

    def is_contiguous(self):
        return self.strides is None


def _calls(s3b, change=None):
    """An engine without a GPU, and each call with the tensors that it takes; change: {name: tensor} in place of good ones."""
    change = change or {}

    def t(name, dtype, *shape):
        return change.get(name) or _Strided(0, dtype, *shape)
    engine = s3b.Engine.__new__(s3b.Engine)
    engine._L, engine.device, engine.h = _Library(), 0, None
    cache = s3b.KVCache(2, PAGES, PAGE, KV, D, data=t("cache", torch.uint8, s3b.kv_cache_bytes(2, KV, D, PAGE, PAGES)))
    bounds = s3b.KVBounds.__new__(s3b.KVBounds)
    bounds.device, bounds.heads, bounds.d, bounds.ref = (1 if "bounds" in change else 0), KV, D, None
    q, out = t("q", torch.float16, 1, 5, 4, D), t("out", torch.float16, 1, 5, 4, D)
    pages, lengths, selected = t("pages", torch.int32, 1, PAGES), t("lengths", torch.int32, 1), t("selected", torch.int32, 1, 3, KV, KEEP)
    lse, scores = t("lse", torch.float32, 1, 5, 4), t("scores", torch.float32, 1, 3, KV, PAGES)
    weights, kept = t("weights", torch.float32, 1, KV, PAGES * PAGE), t("kept", torch.int32, 1, KV, 40)
    weights_out, pages_out, lengths_out = t("weights_out", torch.float32, 1, KV, 40), t("pages_out", torch.int32, 1, 3), t("lengths_out", torch.int32, 1)
    return engine, [
        (("cache", "bounds", "pages", "lengths"), lambda: engine.cache_bounds(cache, bounds, pages, lengths)),
        (("bounds", "q", "selected", "pages", "lengths", "scores"), lambda: engine.cache_select(bounds, q, selected, pages, lengths, share=2, scores=scores)),
        (("cache", "q", "out", "selected", "pages", "lengths", "lse"),
         lambda: engine.cache_attention_selected(cache, q, out, selected, pages, lengths, 0.1, share=2, lse=lse)),
        (("cache", "q", "lse", "weights", "pages", "lengths"), lambda: engine.cache_weights(cache, q, lse, weights, pages, lengths, 0.1)),
        (("cache", "weights", "pages", "lengths", "pages_out", "lengths_out", "kept", "weights_out"),
         lambda: engine.cache_evict(cache, weights, pages, lengths, pages_out, lengths_out, kept, weights_out=weights_out))]


def _check(s3b, name, tensor):
    engine, calls = _calls(s3b, {} if name is None else {name: tensor})
    met = 0
    for names, call in calls:
        before = engine._L.calls
        if name in names:
            met += 1
            with pytest.raises(s3b.S3BError):
                call()
            assert engine._L.calls == before
        elif name != "cache":
            call()
            assert engine._L.calls == before + 1
    assert met or name is None


def test_good_tensors_pass(s3b):
    _check(s3b, None, None)


SHAPES = {"q": (torch.float16, 1, 5, 4, D), "out": (torch.float16, 1, 5, 4, D), "pages": (torch.int32, 1, PAGES), "lengths": (torch.int32, 1),
          "selected": (torch.int32, 1, 3, KV, KEEP), "lse": (torch.float32, 1, 5, 4), "scores": (torch.float32, 1, 3, KV, PAGES),
          "weights": (torch.float32, 1, KV, PAGES * PAGE), "kept": (torch.int32, 1, KV, 40), "weights_out": (torch.float32, 1, KV, 40),
          "pages_out": (torch.int32, 1, 3), "lengths_out": (torch.int32, 1), "cache": (torch.uint8, 1 << 20), "bounds": (torch.int8, 1)}


@pytest.mark.parametrize("name", sorted(SHAPES))
def test_tensors_of_another_gpu_are_refused(s3b, name):
    _check(s3b, name, _Strided(1, *SHAPES[name]))


@pytest.mark.parametrize("name", sorted(set(SHAPES) - {"cache", "bounds"}))
def test_other_types_and_shapes_are_refused(s3b, name):
    dtype, *shape = SHAPES[name]
    other = torch.int64 if dtype is torch.int32 else torch.bfloat16
    _check(s3b, name, _Strided(0, other, *shape))
    _check(s3b, name, _Strided(0, dtype, *shape, 1))
    if len(shape) > 1:
        _check(s3b, name, _Strided(0, dtype, 2, *shape[1:]))


@pytest.mark.parametrize("name,shape,strides", [
    ("q", (1, 5, 4, D), (1280, 256, 64, 2)), ("out", (1, 5, 4, D), (1280, 256, 64, 2)), ("selected", (1, 3, KV, KEEP), (0, 9, 3, 1)),
    ("lse", (1, 5, 4), (20, 1, 5)), ("weights", (1, KV, PAGES * PAGE), (1, 1, 2)), ("kept", (1, KV, 40), (80, 41, 1)), ("weights_out", (1, KV, 40), (80, 41, 1)),
    ("scores", (1, 3, KV, PAGES), (24, 8, 4, 2)), ("pages", (1, PAGES), (8, 2))])
def test_strides_are_refused(s3b, name, shape, strides):
    _check(s3b, name, _Strided(0, SHAPES[name][0], *shape, strides=strides))


@pytest.mark.parametrize("name,shape", [("weights", (1, KV, PAGES * PAGE - 1)), ("pages_out", (1, 2)), ("selected", (1, 5, KV, KEEP)), ("selected", (1, 3, 4, KEEP)),
                                        ("q", (1, 5, 4, 128)), ("weights", (1, 4, PAGES * PAGE))])
def test_sizes_that_do_not_fit_are_refused(s3b, name, shape):
    _check(s3b, name, _Strided(0, SHAPES[name][0], *shape))


@pytest.mark.parametrize("wrong", [dict(window=1 << 40, causal=True), dict(share=0), dict(share=-1), dict(sink=2, recent=2), dict(sink=-1), dict(recent=-1), dict(sink=1 << 40)])
def test_numbers_out_of_range_are_refused(s3b, wrong):
    engine, _ = _calls(s3b)
    cache = s3b.KVCache(2, PAGES, PAGE, KV, D, data=_Strided(0, torch.uint8, s3b.kv_cache_bytes(2, KV, D, PAGE, PAGES)))
    bounds = s3b.KVBounds.__new__(s3b.KVBounds)
    bounds.device, bounds.heads, bounds.d, bounds.ref = 0, KV, D, None
    q, pages, lengths = _Strided(0, torch.float16, 1, 5, 4, D), _Strided(0, torch.int32, 1, PAGES), _Strided(0, torch.int32, 1)
    args = dict(share=2, sink=0, recent=1)
    args.update(wrong)
    with pytest.raises(s3b.S3BError):
        engine.cache_select(bounds, q, _Strided(0, torch.int32, 1, 3, KV, KEEP), pages, lengths, **args)
    if "sink" in wrong or "recent" in wrong:
        with pytest.raises(s3b.S3BError):
            engine.cache_evict(cache, _Strided(0, torch.float32, 1, KV, PAGES * PAGE), pages, lengths, _Strided(0, torch.int32, 1, 3), _Strided(0, torch.int32, 1),
                               _Strided(0, torch.int32, 1, KV, 3), **wrong)
    assert engine._L.calls == 0


@pytest.mark.parametrize("scale", [1e300, -1e300])
def test_a_scale_that_is_no_f32_is_refused(s3b, scale):
    engine, _ = _calls(s3b)
    cache = s3b.KVCache(2, PAGES, PAGE, KV, D, data=_Strided(0, torch.uint8, s3b.kv_cache_bytes(2, KV, D, PAGE, PAGES)))
    q, pages, lengths = _Strided(0, torch.float16, 1, 5, 4, D), _Strided(0, torch.int32, 1, PAGES), _Strided(0, torch.int32, 1)
    with pytest.raises(s3b.S3BError):
        engine.cache_attention_selected(cache, q, q, _Strided(0, torch.int32, 1, 3, KV, KEEP), pages, lengths, scale, share=2)
    with pytest.raises(s3b.S3BError):
        engine.cache_weights(cache, q, _Strided(0, torch.float32, 1, 5, 4), _Strided(0, torch.float32, 1, KV, PAGES * PAGE), pages, lengths, scale)
    assert engine._L.calls == 0
