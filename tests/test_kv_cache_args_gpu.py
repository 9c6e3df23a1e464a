"""Arguments of the quantised cache's calls at their limits: what is refused before any kernel runs, and what has to be taken."""
import ctypes

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture
def call(s3b, engine):
    """s3b_op_cache_attention over a cache of 4 pages of 16 tokens, 2 heads of 64, with one query of 4 heads; arguments by name.
    Returns the status."""
    cache = s3b.KVCache(2, 4, 16, 2, 64)
    k = torch.ones(64, 2, 64, device="cuda")
    engine.cache_write(cache, k, k, torch.arange(64, device="cuda"))
    t = dict(q=torch.ones(2, 1, 4, 64, device="cuda", dtype=torch.float16), out=torch.zeros(2, 1, 4, 64, device="cuda"),
             lse=torch.zeros(2, 1, 4, device="cuda"), pages=torch.arange(8, dtype=torch.int32, device="cuda") % 4,
             lengths=torch.full((4,), 64, dtype=torch.int32, device="cuda"))

    def go(batch=1, page_size=16, max_pages=4, stride=4, scale=0.125, offset=(), **kw):
        at = {n: x.data_ptr() + dict(offset).get(n, 0) for n, x in t.items()}
        desc = s3b.KVCacheDesc(2, 2, 64, page_size, 4 * 16 // page_size if page_size <= 64 else 1, cache.data.data_ptr())
        return engine._L.s3b_op_cache_attention(engine.h, ctypes.byref(desc), at["q"], 256, 256, 64, at["out"], 1, 256, 256, 64, at["lse"],
                                                at["pages"], stride, max_pages, at["lengths"], batch, 1, 4, scale, 0, 0)
    go.tensors = t
    yield go
    engine.sync()


@pytest.mark.parametrize("page_size,max_pages", [(16, (1 << 27) - 1), (16, (1 << 27) - 511), (64, (1 << 25) - 127), (2 ** 31 - 16, 1)])
def test_refuses_page_tables_of_too_many_tokens(call, page_size, max_pages):
    """Past 2^31 - 8192 tokens the kernels' 32-bit token numbers would wrap."""
    assert call(page_size=page_size, max_pages=max_pages, stride=max_pages) == -6


def test_takes_page_tables_of_nearly_2_to_31_tokens(call, engine):
    """The width of the table alone costs nothing: the length says what is read."""
    assert call(max_pages=(1 << 27) - 512, stride=1 << 27) == 0
    engine.sync()
    assert (call.tensors["out"][0] == 1).all()


@pytest.mark.parametrize("scale", [2.0 ** 57, 1e20, 3e38])
def test_refuses_scales_past_the_scores_range(call, scale):
    """Scores of -1e30 and less would count as none at all, and the row as one that sees nothing."""
    assert call(scale=scale) == -1


@pytest.mark.parametrize("nq", [1, 140])
def test_largest_scale(s3b, engine, nq):
    """Every score far below zero: the row still takes the largest."""
    cache = s3b.KVCache(8, 2, 16, 1, 64)
    k = -100.0 * torch.ones(32, 1, 64, device="cuda")
    k[17] = -90.0
    v = torch.arange(32, device="cuda", dtype=torch.float32)[:, None, None].expand(32, 1, 64).contiguous()
    engine.cache_write(cache, k, v, torch.arange(32, device="cuda"))
    q = torch.full((1, nq, 1, 64), 6e4, device="cuda", dtype=torch.float16)
    out = torch.empty(q.shape, device="cuda")
    engine.cache_attention(cache, q, out, torch.arange(2, dtype=torch.int32, device="cuda")[None],
                           torch.tensor([32], dtype=torch.int32, device="cuda"), 2.0 ** 56)
    engine.sync()
    assert (out - 17).abs().max() < 17 * 2.0 ** -10


@pytest.mark.parametrize("name,offset", [("pages", 2), ("lengths", 1), ("lse", 2), ("q", 8), ("out", 4)])
def test_refuses_pointers_off_their_size(call, name, offset):
    assert call(offset=[(name, offset)], max_pages=3) == -1


def test_refuses_slots_off_their_size(s3b, engine):
    cache = s3b.KVCache(2, 1, 16, 1, 64)
    rows, slots = torch.zeros(2, 1, 64, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    k, at = rows.data_ptr(), slots.data_ptr() + 4
    assert engine._L.s3b_op_cache_write(engine.h, cache.ref, k, 64, 64, k, 64, 64, 0, at, 2) == -1
    assert engine._L.s3b_op_cache_read(engine.h, cache.ref, at, 2, k, 64, 64, None, 0, 0, 0) == -1
    engine.sync()


@pytest.mark.parametrize("nq", [1, 300])
def test_one_page_row_for_all_sequences(s3b, engine, nq):
    """A row of the page table expanded over the batch, as sequences over one cache have it."""
    g = torch.Generator(device="cuda").manual_seed(nq)
    cache = s3b.KVCache(2, 9, 16, 2, 64)
    k, v = (torch.randn(144, 2, 64, device="cuda", generator=g) for _ in "kv")
    engine.cache_write(cache, k, v, torch.arange(144, device="cuda"))
    row = torch.randperm(9, device="cuda", generator=g).to(torch.int32)[None]
    q = torch.randn(5, nq, 4, 64, device="cuda", generator=g).half()
    lens = torch.tensor([144, 0, 100, 17, 1], dtype=torch.int32, device="cuda")
    a, b = torch.empty_like(q), torch.empty_like(q)
    engine.cache_attention(cache, q, a, row.expand(5, -1), lens, 0.125)
    engine.cache_attention(cache, q, b, row.repeat(5, 1), lens, 0.125)
    engine.sync()
    assert torch.equal(a, b)


def test_strides_of_one_entry_mean_nothing(s3b, engine):
    g = torch.Generator(device="cuda").manual_seed(2)
    cache = s3b.KVCache(8, 4, 16, 1, 64)
    k, v = (torch.randn(1, 1, 64, device="cuda", generator=g) for _ in "kv")
    slots = torch.arange(40, 44, device="cuda")[::4]
    assert slots.shape == (1,) and slots.stride() == (4,)
    engine.cache_write(cache, k, v, slots)
    q = torch.randn(1, 1, 1, 64, device="cuda", generator=g).half()
    out = torch.empty(1, 1, 1, 64, device="cuda")
    kept = torch.empty(1, 1, 64, device="cuda")
    engine.cache_read(cache, slots, None, kept)
    engine.cache_write(cache, k, v, torch.tensor([32], device="cuda"))
    pages, lens = torch.tensor([[2, 7]], dtype=torch.int32, device="cuda")[:, ::2], torch.ones(3, dtype=torch.int32, device="cuda")[::3]
    engine.cache_attention(cache, q, out, pages, lens, 0.125)
    engine.sync()
    assert (out[0, 0] - kept[0]).abs().max() <= 2.0 ** -10 * kept.abs().max()


def test_refuses_page_rows_that_overlap(call):
    assert call(batch=2, stride=3) == -1
    assert call(batch=2, stride=-4) == -1
