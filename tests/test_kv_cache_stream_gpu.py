"""The quantised key / value cache's kernels in a stream: each may take its place while its predecessor runs, so what one writes
and the next reads is tested without a wait of the host between them."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qtype,d,dtype", [(2, 128, torch.float16), (3, 256, torch.float16), (8, 64, torch.float32)])
def test_calls_see_what_their_predecessors_wrote(s3b, engine, qtype, d, dtype):
    """Read, overwrite the same slots, read, attend with few and with many rows, over and over, the calls back to back: every
    result has to be, bit for bit, that of the same calls with a sync after each."""
    g = torch.Generator(device="cuda").manual_seed(d)
    n, heads, page, rounds = 3000, 2, 16, 12
    cache = s3b.KVCache(qtype, 200, page, heads, d)
    table = torch.randperm(200, device="cuda", generator=g).to(torch.int32)[None, :188].contiguous()
    at = torch.arange(n, device="cuda")
    slots = table[0].long()[at // page] * page + at % page
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    rows = [[torch.randn(n, heads, d, device="cuda", generator=g).to(dtype) for _ in "kv"] for _ in range(rounds)]
    queries = [torch.randn(1, nq, 4, d, device="cuda", generator=g).half() for nq in (1, 300)]

    def new(count, *shape):
        return [torch.full(shape, 3.0, device="cuda", dtype=torch.float16) for _ in range(count)]

    def go(wait):
        cache.data.zero_()
        outs = [new(4, n, heads, d) + [torch.empty_like(q) for q in queries] + [torch.empty_like(queries[0])] for _ in rows]
        torch.cuda.synchronize()
        for (k, v), (k0, v0, k1, v1, few, many, fed) in zip(rows, outs):
            for call in (lambda: engine.cache_read(cache, slots, k0, v0),
                         lambda: engine.cache_write(cache, k, v, slots),
                         lambda: engine.cache_read(cache, slots, k1, v1),
                         lambda: engine.cache_attention(cache, queries[0], few, table, lens, d ** -0.5),
                         lambda: engine.cache_attention(cache, queries[1], many, table, lens, d ** -0.5),
                         # a query that the call before has written
                         lambda: engine.cache_attention(cache, few, fed, table, lens, d ** -0.5)):
                call()
                if wait:
                    engine.sync()
        engine.sync()
        return outs

    waited, queued = go(True), go(False)
    for i, (a, b) in enumerate(zip(waited, queued)):
        for x, y in zip(a, b):
            assert torch.equal(x, y), i
    # each round reads first what the round before wrote, then its own
    for before, after in zip(queued, queued[1:]):
        assert torch.equal(before[2], after[0]) and torch.equal(before[3], after[1])
        assert not torch.equal(after[0], after[2])


def test_calls_see_indexes_made_on_the_device(s3b, engine):
    """Slots, page table, lengths and rows of a call come from kernels just before it."""
    g = torch.Generator(device="cuda").manual_seed(1)
    d, page, pages = 64, 16, 40
    cache = s3b.KVCache(8, pages, page, 1, d)
    n = pages * page
    got = []
    for wait in (True, False):
        cache.data.zero_()
        g.manual_seed(7)
        outs = []
        for i in range(8):
            table = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)[None]
            at = torch.arange(n, device="cuda")
            slots = table[0].long()[at // page] * page + at % page
            k, v = (torch.randn(n, 1, d, device="cuda", generator=g) for _ in "kv")
            q = torch.randn(1, 1 + 140 * (i % 2), 1, d, device="cuda", generator=g).half()
            lens = torch.full((1,), n - i, dtype=torch.int32, device="cuda")
            out = torch.empty_like(q)
            if wait:
                engine.sync()
            engine.cache_write(cache, k, v, slots)
            if wait:
                engine.sync()
            engine.cache_attention(cache, q, out, table, lens, 0.125)
            if wait:
                engine.sync()
            outs.append(out)
        engine.sync()
        got.append(outs)
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("qtype,d,heads,kv,nq", [(8, 256, 1, 1, 30), (8, 256, 2, 1, 300), (8, 128, 8, 2, 40), (8, 128, 2, 2, 130),
                                                 (3, 256, 2, 2, 60), (2, 128, 4, 1, 64)])
def test_many_rows_while_the_cache_arrives_unevenly(s3b, engine, qtype, d, heads, kv, nq):
    """Pages of 16 tokens spread over 2 GiB of memory that this call touches for the first time since another buffer was cleared,
    so that the copies of a tile's halves land apart and out of order: every repetition has to give the same, and what the same
    tokens give from a small cache in order."""
    g = torch.Generator(device="cuda").manual_seed(d)
    n, page = 20000, 16
    at = torch.arange(n, device="cuda")
    k, v = (torch.randn(n, kv, d, device="cuda", generator=g).half() for _ in "kv")
    q = torch.randn(1, nq, heads, d, device="cuda", generator=g).half()
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    flush = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    outs = []
    for total in (n // page, (2 << 30) // s3b.kv_cache_bytes(qtype, kv, d, page, 1)):
        cache = s3b.KVCache(qtype, total, page, kv, d, data=torch.full((s3b.kv_cache_bytes(qtype, kv, d, page, total),), 0xFF,
                                                                       dtype=torch.uint8, device="cuda"))
        table = torch.arange(total, device="cuda") if not outs else torch.randperm(total, device="cuda", generator=g)
        table = table[:n // page].to(torch.int32)[None].contiguous()
        engine.cache_write(cache, k, v, table[0].long()[at // page] * page + at % page)
        for _ in range(1 if not outs else 12):
            flush.zero_()
            out = torch.empty_like(q)
            engine.cache_attention(cache, q, out, table, lens, d ** -0.5)
            outs.append(out)
        engine.sync()
    assert torch.isfinite(outs[0]).all()
    for out in outs[1:]:
        assert torch.equal(out, outs[0])


@pytest.fixture
def captured(s3b):
    """An engine of its own on a stream of its own, and a function that runs a call under capture and returns the graph."""
    stream = torch.cuda.Stream()
    own = s3b.Engine(0)
    own.set_stream(stream.cuda_stream)

    def capture(call):
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            call()
        return graph
    yield own, stream, capture
    torch.cuda.synchronize()
    own.close()


def _filled(s3b, engine, qtype, n, heads, d, page=16):
    g = torch.Generator(device="cuda").manual_seed(n)
    cache = s3b.KVCache(qtype, -(-n // page), page, heads, d)
    k, v = (torch.randn(n, heads, d, device="cuda", generator=g).half() for _ in "kv")
    engine.cache_write(cache, k, v, torch.arange(n, device="cuda"))
    engine.sync()
    return cache, torch.arange(-(-n // page), dtype=torch.int32, device="cuda")[None], torch.tensor([n], dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("nq,qtype,d", [(1, 2, 128), (6, 3, 64), (70, 8, 128), (900, 2, 256)])
def test_graph_survives_a_larger_call(s3b, engine, captured, nq, qtype, d):
    """A captured call, replayed with new queries before and after calls that need a larger workspace, which has to be another
    buffer than the graph's."""
    own, stream, capture = captured
    cache, pages, lens = _filled(s3b, engine, qtype, 3000, 2, d)
    big = _filled(s3b, engine, 2, 30000, 2, d)
    g = torch.Generator(device="cuda").manual_seed(nq)
    q = torch.randn(1, nq, 8, d, device="cuda", generator=g).half()
    out, ref = torch.empty_like(q), torch.empty_like(q)
    torch.cuda.synchronize()
    own.cache_attention(cache, q, out, pages, lens, d ** -0.5)  # the shape once
    own.sync()
    graph = capture(lambda: own.cache_attention(cache, q, out, pages, lens, d ** -0.5))

    def check():
        q.copy_(torch.randn(q.shape, device="cuda", generator=g))
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        engine.cache_attention(cache, q, ref, pages, lens, d ** -0.5)
        engine.sync()
        assert torch.equal(out, ref)
    check()
    many = torch.randn(1, 5000, 8, d, device="cuda", generator=g).half()
    wide = torch.randn(20000, 1, 2, d, device="cuda", generator=g).half()
    torch.cuda.synchronize()
    for big_q, rows in ((many, 1), (wide, len(wide))):  # more rows, then more sequences
        got, again = torch.empty_like(big_q), torch.empty_like(big_q)
        torch.cuda.synchronize()
        tables, lengths = (t.expand(rows, *t.shape[1:]).contiguous() for t in big[1:])
        lengths = (lengths // (1 if rows == 1 else 100)).contiguous()
        torch.cuda.synchronize()
        own.cache_attention(big[0], big_q, got, tables, lengths, d ** -0.5)
        own.sync()
        engine.cache_attention(big[0], big_q, again, tables, lengths, d ** -0.5)
        engine.sync()
        assert torch.equal(got, again)
        check()
        check()


def test_few_rows_captured_after_many(s3b, engine, captured):
    """A call of few rows is captured when only one of many rows has run: nothing may have to be allocated then."""
    own, stream, capture = captured
    cache, pages, lens = _filled(s3b, engine, 2, 2000, 2, 128)
    many, few = (torch.randn(1, nq, 8, 128, device="cuda").half() for nq in (400, 1))
    outs = [torch.empty_like(x) for x in (many, few, few)]
    torch.cuda.synchronize()
    own.cache_attention(cache, many, outs[0], pages, lens, 0.1)
    own.sync()
    graph = capture(lambda: own.cache_attention(cache, few, outs[1], pages, lens, 0.1))
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    engine.cache_attention(cache, few, outs[2], pages, lens, 0.1)
    engine.sync()
    assert torch.equal(outs[1], outs[2])


def test_growing_during_a_capture_is_refused(s3b, engine, captured):
    """The first call of an engine inside a capture: an error, no allocation, and the capture and the engine go on."""
    own, stream, capture = captured
    cache, pages, lens = _filled(s3b, engine, 2, 2000, 2, 128)
    q = torch.randn(1, 1, 8, 128, device="cuda").half()
    out, ref = torch.empty_like(q), torch.empty_like(q)
    rows = [torch.empty(4, 2, 128, device="cuda", dtype=torch.float16) for _ in "kv"]
    slots = torch.arange(4, device="cuda")

    def call():
        with pytest.raises(s3b.S3BError, match="capture"):
            own.cache_attention(cache, q, out, pages, lens, 0.1)
        own.cache_read(cache, slots, *rows)
    graph = capture(call)
    graph.replay()
    own.cache_attention(cache, q, out, pages, lens, 0.1)
    own.sync()
    engine.cache_attention(cache, q, ref, pages, lens, 0.1)
    engine.sync()
    assert torch.equal(out, ref) and rows[0].any()


@pytest.mark.parametrize("side", [False, True])
def test_new_cache_is_cleared_before_its_first_write(s3b, side):
    """A cache of 4 GiB made on torch's stream (or a side stream) and written at once on the engine's own."""
    own = s3b.Engine(0)
    page, d = 64, 128
    pages = (4 << 30) // s3b.kv_cache_bytes(8, 1, d, page, 1)
    k, v = (torch.randn(64, 1, d, device="cuda") for _ in "kv")
    slots = (pages - 1) * page + torch.arange(64, device="cuda")
    rows = [torch.empty(64, 1, d, device="cuda") for _ in "kv"]
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream() if side else torch.cuda.current_stream()):
        cache = s3b.KVCache(8, pages, page, 1, d)
    own.cache_write(cache, k, v, slots)
    own.sync()
    torch.cuda.synchronize()
    own.cache_read(cache, slots, *rows)
    own.sync()
    own.close()
    for x, y in zip(rows, (k, v)):
        assert (x - y).abs().max() <= y.abs().max() / 127
