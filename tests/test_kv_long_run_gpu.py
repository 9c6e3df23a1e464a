"""Long caches as a program uses them: the calls one after another, without a wait between them, in captured graphs, on other
streams; and what they refuse."""
import ctypes
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


class Stream:
    """One growing sequence, cut down when it passes `most` tokens: `budget` are kept, in a second set of pages that takes turns
    with the first."""

    def __init__(self, s3b, engine, qtype, heads, kv, d, page, most, budget, keep, decay=0.9, seed=0):
        self.s3b, self.engine, self.kv, self.d, self.heads, self.page, self.budget, self.keep, self.decay = s3b, engine, kv, d, heads, page, budget, keep, decay
        per = -(-(most + 64) // page)  # it grows past `most` by one step before it is cut
        self.most = most
        self.cache = s3b.KVCache(qtype, 2 * per, page, kv, d)
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.sets = torch.randperm(2 * per, device="cuda", generator=g).to(torch.int32).view(2, 1, per)
        self.now = 0
        self.bounds = s3b.KVBounds(self.cache)
        self.weights = [torch.zeros(1, kv, per * page, device="cuda") for _ in "ab"]
        self.n = 0
        self.k = torch.zeros(0, kv, d, device="cuda", dtype=torch.float64)  # what the plain computation holds, by head
        self.v, self.w = self.k.clone(), torch.zeros(0, kv, device="cuda", dtype=torch.float64)

    def length(self):
        return torch.tensor([self.n], dtype=torch.int32, device="cuda")

    def pages(self):
        return self.sets[self.now]

    def slots(self, first, n):
        at = torch.arange(first, first + n, device="cuda")
        return self.pages()[0].long()[at // self.page] * self.page + at % self.page

    def append(self, k, v):
        n = len(k)
        slots = self.slots(self.n, n)
        self.engine.cache_write(self.cache, k, v, slots)
        self.n += n
        self.engine.cache_bounds(self.cache, self.bounds, self.pages(), self.length(), new=n)
        held = [torch.empty(n, self.kv, self.d, device="cuda") for _ in "kv"]
        self.engine.cache_read(self.cache, slots, *held)
        self.k, self.v = torch.cat([self.k, held[0].double()]), torch.cat([self.v, held[1].double()])
        self.w = torch.cat([self.w, torch.zeros(n, self.kv, device="cuda", dtype=torch.float64)])

    def attend(self, q):
        """Attention over the chosen pages, and the weights that all tokens gain; the plain results beside it."""
        nq, scale = q.shape[1], self.d ** -0.5
        selected = torch.empty(1, nq, self.kv, self.keep, dtype=torch.int32, device="cuda")
        out, dense = torch.empty(q.shape, device="cuda"), torch.empty(q.shape, device="cuda")
        lse = torch.empty(q.shape[:3], device="cuda")
        self.engine.cache_select(self.bounds, q, selected, self.pages(), self.length(), sink=1, recent=1, causal=True)
        self.engine.cache_attention_selected(self.cache, q, out, selected, self.pages(), self.length(), scale, causal=True)
        self.engine.cache_attention(self.cache, q, dense, self.pages(), self.length(), scale, causal=True, lse=lse)
        self.engine.cache_weights(self.cache, q, lse, self.weights[self.now], self.pages(), self.length(), scale, decay=self.decay, causal=True)
        # plain
        group, at = self.heads // self.kv, torch.arange(self.n, device="cuda")
        want = torch.zeros(q.shape, device="cuda", dtype=torch.float64)
        self.w *= self.decay
        for h in range(self.heads):
            z = q[0, :, h].double() @ self.k[:, h // group].T * scale
            hide = at[None] >= self.n - nq + 1 + torch.arange(nq, device="cuda")[:, None]
            self.w[:, h // group] += z.masked_fill(hide, -math.inf).softmax(-1).sum(0)
            for i in range(nq):
                names = selected[0, i, h // group]
                inside = torch.isin(at // self.page, names[names >= 0]) & ~hide[i]
                want[0, i, h] = z[i].masked_fill(~inside, -math.inf).softmax(-1) @ self.v[:, h // group]
        return out, want, selected

    def cut(self):
        """Evicts where the sequence has grown past `most`. Returns whether."""
        if self.n <= self.most:
            return False
        kept = torch.empty(1, self.kv, self.budget, dtype=torch.int32, device="cuda")
        n_out = torch.empty(1, dtype=torch.int32, device="cuda")
        other = 1 - self.now
        w_out = torch.empty(1, self.kv, self.budget, device="cuda")
        self.engine.cache_evict(self.cache, self.weights[self.now], self.pages(), self.length(), self.sets[other], n_out, kept, sink=2, recent=8,
                                weights_out=w_out)
        self.weights[other].zero_()
        self.weights[other][:, :, :self.budget] = w_out
        self.now, self.n = other, self.budget
        self.engine.cache_bounds(self.cache, self.bounds, self.pages(), n_out)
        at = kept[0].long().T                                             # [budget, heads]
        head = torch.arange(self.kv, device="cuda")
        weights = self.w[at, head]
        # the kept are the heaviest, up to what f32 sums differ
        least = weights[2:-8].amin(0)
        gone = self.w.clone()
        gone[at, head] = -1
        assert (gone.amax(0) <= least + 1e-5 * least.abs() + 1e-9).all()
        assert (at[:2] == torch.arange(2, device="cuda")[:, None]).all() and (at[1:] > at[:-1]).all()
        self.k, self.v, self.w = self.k[at, head], self.v[at, head], weights
        return True


@pytest.mark.parametrize("qtype,heads,kv,d,page", [(2, 4, 2, 64, 16), (3, 3, 1, 128, 48), (8, 2, 2, 256, 32)])
def test_stream(s3b, engine, qtype, heads, kv, d, page):
    """A prompt, then single tokens and drafts, cut several times: every step's output against the plain computation on what is
    left."""
    g = torch.Generator(device="cuda").manual_seed(qtype)
    st = Stream(s3b, engine, qtype, heads, kv, d, page, most=400, budget=200, keep=5, seed=qtype)
    cuts = 0
    for step, n in enumerate([350] + [1, 1, 5, 40] * 16):
        rows = [torch.randn(n, kv, d, device="cuda", generator=g) for _ in "kv"]
        st.append(*rows)
        q = torch.randn(1, min(n, 5), heads, d, device="cuda", generator=g).half()
        out, want, selected = st.attend(q)
        engine.sync()
        assert ((out.double() - want).norm() <= 2.0 ** -11 * 1.5 * want.norm()), step
        assert (selected[..., :5] >= 0).all() or st.n < 5 * page
        w = st.weights[st.now][0, :, :st.n].T
        assert (w.double() - st.w).abs().max() <= 1e-5 * st.w.max() + 1e-7
        cuts += st.cut()
    assert cuts >= 3


def _world(s3b, engine, qtype=2, d=64, kv=2, heads=4, n=3000, page=16, seed=0, batch=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    per = -(-n // page)
    cache = s3b.KVCache(qtype, 2 * batch * per, page, kv, d)
    k, v = (torch.randn(batch * per * page, kv, d, device="cuda", generator=g).half() for _ in "kv")
    engine.cache_write(cache, k, v, torch.arange(batch * per * page, device="cuda"))
    engine.sync()
    return dict(cache=cache, bounds=s3b.KVBounds(cache), pages=torch.arange(batch * per, dtype=torch.int32, device="cuda").view(batch, per),
                lengths=torch.full((batch,), n, dtype=torch.int32, device="cuda"),
                pages_out=torch.arange(batch * per, 2 * batch * per, dtype=torch.int32, device="cuda").view(batch, per),
                q=torch.randn(batch, 3, heads, d, device="cuda", generator=g).half())


def _outs(w, keep=20, tokens=500):
    batch, nq, heads, d = w["q"].shape
    kv = w["cache"].heads
    return dict(selected=torch.zeros(batch, nq, kv, keep, dtype=torch.int32, device="cuda"), out=torch.zeros_like(w["q"]),
                lse=torch.zeros(batch, nq, heads, device="cuda"), weights=torch.ones(batch, kv, w["pages"].shape[1] * w["cache"].page_size, device="cuda"),
                kept=torch.zeros(batch, kv, tokens, dtype=torch.int32, device="cuda"), lengths_out=torch.zeros(batch, dtype=torch.int32, device="cuda"),
                weights_out=torch.zeros(batch, kv, tokens, device="cuda"), again=torch.zeros_like(w["q"]), codes=None)


def _calls(e, w, o):
    """All calls, each on what those before it have written."""
    scale = w["q"].shape[-1] ** -0.5
    return [lambda: e.cache_bounds(w["cache"], w["bounds"], w["pages"], w["lengths"]),
            lambda: e.cache_select(w["bounds"], w["q"], o["selected"], w["pages"], w["lengths"], sink=1, recent=2, causal=True),
            lambda: e.cache_attention_selected(w["cache"], w["q"], o["out"], o["selected"], w["pages"], w["lengths"], scale, causal=True, lse=o["lse"]),
            lambda: e.cache_weights(w["cache"], o["out"], o["lse"], o["weights"], w["pages"], w["lengths"], scale, decay=0.5),
            lambda: e.cache_evict(w["cache"], o["weights"], w["pages"], w["lengths"], w["pages_out"], o["lengths_out"], o["kept"], recent=3,
                                  weights_out=o["weights_out"]),
            lambda: e.cache_bounds(w["cache"], w["bounds"], w["pages_out"], o["lengths_out"]),
            lambda: e.cache_select(w["bounds"], o["out"], o["selected"], w["pages_out"], o["lengths_out"]),
            lambda: e.cache_attention_selected(w["cache"], o["out"], o["again"], o["selected"], w["pages_out"], o["lengths_out"], scale)]


@pytest.mark.parametrize("qtype,d,n", [(2, 64, 3000), (3, 128, 9000), (8, 256, 700), (2, 128, 20000)])
def test_calls_see_what_their_predecessors_wrote(s3b, engine, qtype, d, n):
    """The calls back to back, over and over with other queries: bit for bit what they give with a wait after each."""
    w = _world(s3b, engine, qtype, d, n=n)
    g = torch.Generator(device="cuda").manual_seed(1)
    queries = [torch.randn(w["q"].shape, device="cuda", generator=g).half() for _ in range(6)]
    got = []
    for wait in (True, False):
        w["bounds"].codes.zero_()
        outs = [_outs(w) for _ in queries]
        torch.cuda.synchronize()
        for q, o in zip(queries, outs):
            w["q"].copy_(q)
            for call in _calls(engine, w, o):
                call()
                if wait:
                    engine.sync()
        engine.sync()
        got.append(outs)
    for a, b in zip(*got):
        for name in a:
            assert a[name] is None or torch.equal(a[name], b[name]), name
    assert not torch.equal(got[0][0]["kept"], got[0][1]["kept"])


@pytest.fixture
def captured(s3b):
    """An engine of its own on a stream of its own, and a function that captures calls and returns the graph."""
    stream = torch.cuda.Stream()
    own = s3b.Engine(0)
    own.set_stream(stream.cuda_stream)

    def capture(calls):
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            for call in calls:
                call()
        return graph
    yield own, stream, capture
    torch.cuda.synchronize()
    own.close()


def test_graph(s3b, engine, captured):
    """All calls in one graph, replayed with other queries, before and after calls that need larger workspaces."""
    own, stream, capture = captured
    w = _world(s3b, engine, 2, 128, n=9000)
    big = _world(s3b, engine, 2, 64, n=40000, batch=40, heads=8)
    o, r, ob = _outs(w), _outs(w), _outs(big, 300, 2000)
    torch.cuda.synchronize()
    for call in _calls(own, w, o):
        call()
    own.sync()
    graph = capture(_calls(own, w, o))
    g = torch.Generator(device="cuda").manual_seed(3)
    for again in range(3):
        w["q"].copy_(torch.randn(w["q"].shape, device="cuda", generator=g))
        for x in (o, r):
            x["weights"].fill_(1.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = {name: x.clone() for name, x in o.items() if x is not None}
        for call in _calls(engine, w, r):
            call()
        engine.sync()
        for name in got:
            assert torch.equal(got[name], r[name]), (again, name)
        for call in _calls(own, big, ob):
            call()
        own.sync()


def test_growing_during_a_capture_is_refused(s3b, engine, captured):
    own, stream, capture = captured
    w = _world(s3b, engine)
    o, r = _outs(w), _outs(w)
    bounds, select, attend, weights, evict = _calls(own, w, o)[:5]

    def refused():
        with pytest.raises(s3b.S3BError, match="capture"):
            attend()
    graph = capture([bounds, select, refused, weights, evict])  # what needs no workspace goes on
    graph.replay()
    torch.cuda.synchronize()
    for call in (bounds, select, attend):
        call()
    own.sync()
    for call in _calls(engine, w, r)[:3]:
        call()
    engine.sync()
    assert torch.equal(o["out"], r["out"]) and torch.equal(o["selected"], r["selected"])


def test_own_stream(s3b, engine):
    """An engine on its own stream, inputs made and waited for on torch's."""
    w = _world(s3b, engine)
    own = s3b.Engine(0)
    o, r = _outs(w), _outs(w)
    torch.cuda.synchronize()
    for call in _calls(own, w, o):
        call()
    own.sync()
    for call in _calls(engine, w, r):
        call()
    engine.sync()
    own.close()
    for name in o:
        assert o[name] is None or torch.equal(o[name], r[name]), name


# ---------------------------------------------------------------- indexes in device memory
def _errors(s3b, engine):
    with pytest.raises(s3b.S3BError, match="out of range"):
        engine.sync()
    engine.sync()


@pytest.mark.parametrize("bad", ["page", "negative page", "length", "negative length"])
def test_bad_indexes(s3b, engine, bad):
    """A page outside the cache, a length past the table: an error at the next sync, nothing read or written outside."""
    w = _world(s3b, engine, n=300)
    for i in range(5):
        o = _outs(w, 4, 50)
        calls = _calls(engine, w, o)[:5]
        for call in calls[:i]:
            call()
        engine.sync()
        pages, lengths = w["pages"].clone(), w["lengths"].clone()
        if "page" in bad:
            w["pages"][0, :] = w["cache"].n_pages if bad == "page" else -1
        else:
            w["lengths"][:] = 305 if bad == "length" else -1
        calls[i]()
        _errors(s3b, engine)
        w["pages"].copy_(pages)
        w["lengths"].copy_(lengths)
        torch.cuda.synchronize()


def test_bad_entry_and_new_page(s3b, engine):
    w = _world(s3b, engine, n=300)
    o = _outs(w, 4, 50)
    calls = _calls(engine, w, o)
    for call in calls[:4]:
        call()
    engine.sync()
    good = o["out"].clone()
    o["selected"][0, :, :, 3] = w["pages"].shape[1]
    calls[2]()
    _errors(s3b, engine)
    selected = o["selected"].clone()
    o["selected"][0, :, :, 3] = -1
    bad = o["out"].clone()
    calls[2]()
    engine.sync()
    assert torch.equal(o["out"], bad) and not torch.equal(o["out"], good)
    data = w["cache"].data.clone()
    w["pages_out"][0, :] = torch.tensor([w["cache"].n_pages, -1], device="cuda").repeat(20)[:w["pages_out"].shape[1]]
    calls[4]()
    _errors(s3b, engine)
    assert torch.equal(w["cache"].data, data) and selected.shape == o["selected"].shape


# ---------------------------------------------------------------- refusals
@pytest.fixture
def raw(s3b, engine):
    """The C calls over one small cache, arguments by name."""
    w = _world(s3b, engine, n=300)
    o = _outs(w, 4, 50)
    L, h = engine._L, engine.h
    d, max_pages = 64, w["pages"].shape[1]

    def at(t, off=0):
        return t.data_ptr() + off if t is not None else 0

    def the_call(pages=w["pages"], stride=max_pages, width=max_pages, lengths=w["lengths"], batch=1, q=w["q"], q_h=d, out=o["out"], lse=o["lse"], sel=o["selected"],
                 keep=4, share=1, nq=3, heads=4, scale=0.1, causal=0, window=0, pages_off=0, q_off=0, out_off=0, lse_off=0):
        return s3b._CALL.pack(at(pages, pages_off), stride, at(lengths), at(q, q_off), 12 * d, 4 * d, q_h, at(out, out_off), 12 * d, 4 * d, d, at(lse, lse_off), at(sel),
                              width, batch, nq, heads, causal, window, keep, share, 0, scale)

    class Calls:
        def bounds(self, recent=5, desc=None, off=0, **kw):
            return L.s3b_op_cache_bounds(h, w["cache"].ref, ctypes.byref(desc) if desc else w["bounds"].ref, the_call(pages_off=off, **kw), recent)

        def select(self, sink=0, recent=0, scores=None, off=0, desc=None, **kw):
            return L.s3b_op_cache_select(h, ctypes.byref(desc) if desc else w["bounds"].ref, the_call(q_off=off, **kw), sink, recent, at(scores) or None)

        def attend(self, off=0, **kw):
            return L.s3b_op_cache_attention_selected(h, w["cache"].ref, the_call(out_off=off, **kw))

        def weights(self, wt=o["weights"], w_b=2 * 16 * max_pages, w_h=16 * max_pages, decay=1.0, off=0, **kw):
            return L.s3b_op_cache_weights(h, w["cache"].ref, the_call(**kw), at(wt, off) or None, w_b, w_h, decay)

        def evict(self, to=None, wt=o["weights"], keep=50, sink=0, recent=0, pages_out=w["pages_out"], stride=max_pages, lengths_out=o["lengths_out"], kept=o["kept"],
                  weights_out=o["weights_out"], off=0, **kw):
            e = s3b._EVICT.pack(ctypes.addressof(to) if to else 0, at(wt), 0, 16 * max_pages, at(pages_out), stride, at(lengths_out), at(kept, off), at(weights_out), keep,
                                sink, recent)
            return L.s3b_op_cache_evict(h, w["cache"].ref, the_call(**kw), e)
    c = Calls()
    c.w, c.o, c.max_pages = w, o, max_pages
    yield c
    engine.sync()


def test_raw_calls_pass(raw, engine):
    assert raw.bounds() == 0 and raw.select() == 0 and raw.attend() == 0 and raw.weights() == 0 and raw.evict() == 0
    assert raw.bounds(batch=0) == 0 and raw.select(batch=0) == 0 and raw.attend(nq=0) == 0 and raw.weights(batch=0) == 0 and raw.evict(batch=0) == 0
    assert raw.bounds(recent=0) == 0 and raw.select(nq=0) == 0
    engine.sync()


@pytest.mark.parametrize("call,args,code", [
    ("bounds", dict(pages=None), -1), ("bounds", dict(lengths=None), -1), ("bounds", dict(batch=2, stride=3), -1), ("bounds", dict(batch=-1), -1), ("bounds", dict(recent=-1), -1),
    ("bounds", dict(width=1 << 27, stride=1 << 27), -6), ("bounds", dict(off=2), -1), ("bounds", dict(width=-1), -1),
    ("select", dict(q=None), -1), ("select", dict(sel=None), -1), ("select", dict(keep=0), -1), ("select", dict(share=0), -1), ("select", dict(sink=3, recent=2), -1),
    ("select", dict(sink=-1), -1), ("select", dict(recent=-1), -1), ("select", dict(heads=3), -1), ("select", dict(heads=0), -1), ("select", dict(window=5), -1),
    ("select", dict(causal=1, window=-1), -1), ("select", dict(q_h=60), -1), ("select", dict(off=8), -1), ("select", dict(nq=-1), -1), ("select", dict(nq=40, share=17), -6),
    ("select", dict(heads=68), -6), ("select", dict(width=1 << 27, stride=1 << 27), -6),
    ("attend", dict(q=None), -1), ("attend", dict(out=None), -1), ("attend", dict(sel=None), -1), ("attend", dict(keep=0), -1), ("attend", dict(share=-2), -1),
    ("attend", dict(scale=0.0), -1), ("attend", dict(scale=-1.0), -1), ("attend", dict(scale=math.nan), -1), ("attend", dict(scale=2.0 ** 57), -1), ("attend", dict(window=1), -1),
    ("attend", dict(off=8), -1), ("attend", dict(heads=5), -1), ("attend", dict(nq=40, share=17), -6), ("attend", dict(keep=1 << 28), -6), ("attend", dict(heads=68), -6),
    ("weights", dict(q=None), -1), ("weights", dict(lse=None), -1), ("weights", dict(wt=None), -1), ("weights", dict(decay=-0.5), -1), ("weights", dict(decay=math.nan), -1),
    ("weights", dict(decay=math.inf), -1), ("weights", dict(w_h=303), -1), ("weights", dict(w_h=0), -1), ("weights", dict(batch=2, w_b=304), -1), ("weights", dict(scale=0.0), -1),
    ("weights", dict(off=2), -1), ("weights", dict(heads=6, nq=1 << 29), -6), ("weights", dict(window=3), -1),
    ("evict", dict(wt=None), -1), ("evict", dict(pages_out=None), -1), ("evict", dict(kept=None), -1), ("evict", dict(lengths_out=None), -1), ("evict", dict(keep=-1), -1),
    ("evict", dict(sink=30, recent=21), -1), ("evict", dict(sink=-1), -1), ("evict", dict(off=2), -1), ("evict", dict(batch=2, stride=3), -1)])
def test_refusals(raw, call, args, code):
    assert getattr(raw, call)(**args) == code


def test_refuses_no_call(engine, raw):
    w, L, h = raw.w, engine._L, engine.h
    assert L.s3b_op_cache_bounds(h, w["cache"].ref, w["bounds"].ref, None, 1) == -1 and L.s3b_op_cache_select(h, w["bounds"].ref, None, 0, 0, None) == -1
    assert L.s3b_op_cache_attention_selected(h, w["cache"].ref, None) == -1 and L.s3b_op_cache_weights(h, w["cache"].ref, None, raw.o["weights"].data_ptr(), 0, 304, 1.0) == -1
    assert L.s3b_op_cache_evict(h, w["cache"].ref, None, None) == -1


def test_refuses_other_shapes(s3b, raw):
    w, o = raw.w, raw.o
    c, b = w["cache"], w["bounds"]
    for heads, d, page, pages in ((1, 64, 16, c.n_pages), (2, 128, 16, c.n_pages), (2, 64, 32, c.n_pages), (2, 64, 16, c.n_pages - 1), (2, 60, 16, c.n_pages), (0, 64, 16, 1)):
        desc = s3b.KVBoundsDesc(heads, d, page, pages, b.codes.data_ptr(), b.steps.data_ptr())
        assert raw.bounds(desc=desc) == -1
    for codes, steps in ((0, b.steps.data_ptr()), (b.codes.data_ptr(), 0), (b.codes.data_ptr() + 8, b.steps.data_ptr()), (b.codes.data_ptr(), b.steps.data_ptr() + 2)):
        desc = s3b.KVBoundsDesc(2, 64, 16, c.n_pages, codes, steps)
        assert raw.bounds(desc=desc) == -1 and raw.select(desc=desc) == -1
    for qtype, heads, d in ((3, 2, 64), (2, 1, 64), (2, 2, 128)):
        assert raw.evict(to=s3b.KVCacheDesc(qtype, heads, d, 16, 4, c.data.data_ptr())) == -1


def test_refuses_arrays_over_each_other(raw):
    w, o = raw.w, raw.o
    assert raw.evict(lengths_out=w["lengths"]) == -1
    assert raw.evict(weights_out=o["weights"]) == -1
    assert raw.evict(weights_out=o["weights"][0, 1, 200:]) == -1
