"""Long caches: bounds of pages, choice of pages, attention over chosen pages, gathered weights, eviction, against plain
implementations in 64 bits on the values that the cache holds (as cache_read gives them, which other tests compare with the host
quantisers). Bounds, scores, choices and moved rows are compared bit for bit.

Tolerances, with u = 2^-11 (half a step of f16): a score's f32 sum over d exact products, scaled block by block, is off by
at most E = (d + 16) 2^-24 scale sum |q| max|k| per row and token. A weight exp(s - m) then by a factor of exp(E) and 2^-21 (ex2),
in numerator and denominator; its product with the block scale is rounded once to f16 (u; what the weight's own rounding leaves is
kept to 2^-22 of it), and the output to its type. In q4_1 a value enters as scale (code - 8) and minimum + 8 scale, each with that
rounding, so |v| counts with the block's largest magnitude and range. Weights far below the largest end in f16's subnormal step,
2^-25 of the largest weight's product with the largest value."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -11
TYPES = [2, 3, 8]


class Sequences:
    """A cache with random keys and values in sequences of the given lengths, over pages in random order; pages that no sequence
    has, and the places behind each sequence's last token, hold 3e4 and -3e4."""

    def __init__(self, s3b, engine, qtype, d, heads, page, lengths, seed=0, spare=2, width=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.g, self.page, self.heads, self.d, self.lens = g, page, heads, d, lengths
        most = max(1, max(-(-n // page) for n in lengths)) if width is None else width
        total = len(lengths) * most + spare
        self.cache = s3b.KVCache(qtype, total, page, heads, d)
        self.pages = torch.randperm(total, device="cuda", generator=g)[:len(lengths) * most].to(torch.int32).view(len(lengths), most)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        n = total * page
        wild = torch.full((n, heads, d), 3e4, device="cuda", dtype=torch.float16)
        wild[:, :, ::2] *= -1
        engine.cache_write(self.cache, wild, wild, torch.arange(n, device="cuda"))
        self.slots = (self.pages.long()[:, :, None] * page + torch.arange(page, device="cuda")).flatten(1)
        k = torch.randn(*self.slots.shape, heads, d, device="cuda", generator=g)
        k = k * torch.exp(0.4 * torch.randn(heads, d, device="cuda", generator=g)) + 0.5 * torch.randn(heads, d, device="cuda", generator=g)
        k += 0.7 * torch.randn(len(lengths), most, 1, heads, d, device="cuda", generator=g).expand(-1, -1, page, -1, -1).flatten(1, 2)
        v = torch.randn(*self.slots.shape, heads, d, device="cuda", generator=g) + 0.3
        for b, m in enumerate(lengths):
            if m:
                engine.cache_write(self.cache, k[b, :m].half(), v[b, :m].half(), self.slots[b, :m].contiguous())
        self.engine = engine

    def queries(self, nq, heads, size=0.8):
        return (size * torch.randn(len(self.lens), nq, heads, self.d, device="cuda", generator=self.g)).half()

    def rows(self, b, dtype=torch.float32):
        """Keys and values of sequence b as the cache holds them."""
        m = self.lens[b]
        k, v = (torch.empty(m, self.heads, self.d, device="cuda", dtype=dtype) for _ in "kv")
        self.engine.cache_read(self.cache, self.slots[b, :m].contiguous(), k, v)
        return k, v


def spans(n, nq, causal, window):
    """[lo, hi) of each query."""
    out = []
    for i in range(nq):
        hi = max(0, n - nq + i + 1) if causal else n
        out.append((max(0, hi - window) if causal and window else 0, hi))
    return out


# ---------------------------------------------------------------- bounds
def plain_bounds(keys, page):
    """Codes [pages, heads, 2, d] and steps [pages, heads] of keys f16 [n, heads, d]."""
    codes, steps = [], []
    for p in keys.double().split(page):
        lo, hi = p.amin(0), p.amax(0)
        peak = torch.maximum(lo.abs(), hi.abs()).amax(-1, keepdim=True)
        inv = torch.where(peak > 0, 127 / peak, 0.0).float().double()
        codes.append(torch.stack([(lo * inv).float().floor().clamp(-127, 127), (hi * inv).float().ceil().clamp(-127, 127)], 1))
        steps.append((peak / 127).float().squeeze(-1))
    return torch.stack(codes).to(torch.int8), torch.stack(steps)


@pytest.mark.parametrize("qtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page,heads,lengths", [(16, 1, [1]), (48, 3, [100, 0, 48, 49]), (64, 2, [700, 63]), (256, 5, [257, 3])])
def test_bounds(s3b, engine, qtype, d, page, heads, lengths):
    q = Sequences(s3b, engine, qtype, d, heads, page, lengths, seed=d + page)
    bounds = s3b.KVBounds(q.cache)
    bounds.codes.fill_(77)
    bounds.steps.fill_(7.0)
    engine.cache_bounds(q.cache, bounds, q.pages, q.lengths)
    engine.sync()
    touched = torch.zeros(q.cache.n_pages, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lengths):
        if not n:
            continue
        codes, steps = plain_bounds(q.rows(b, torch.float16)[0], page)
        at = q.pages[b, :len(codes)].long()
        touched[at] = True
        assert torch.equal(bounds.codes[at], codes) and torch.equal(bounds.steps[at], steps)
        assert torch.equal(bounds.values(at), codes * steps[..., None, None])
        # they bound the keys, up to f32 roundings of the steps
        lo, hi = bounds.values(at).repeat_interleave(page, 0)[:n].unbind(2)
        k = q.rows(b, torch.float16)[0].float()
        slack = steps.repeat_interleave(page, 0)[:n, :, None] * 127 * 2.0 ** -22
        assert (k >= lo - slack).all() and (k <= hi + slack).all()
    assert (bounds.codes[~touched] == 77).all() and (bounds.steps[~touched] == 7).all()


def test_values_of_bounds(s3b, engine):
    """Pages in any order, twice, and outside; none at all; another stream; refusals."""
    cache = s3b.KVCache(2, 9, 16, 3, 128)
    bounds = s3b.KVBounds(cache)
    g = torch.Generator(device="cuda").manual_seed(1)
    bounds.codes.copy_(torch.randint(-127, 128, bounds.codes.shape, device="cuda", generator=g))
    bounds.steps.copy_(torch.rand(bounds.steps.shape, device="cuda", generator=g))
    pages = torch.tensor([8, 0, 3, 3, -1, 9, 1], device="cuda")
    want = bounds.codes[pages.clamp(0, 8)] * bounds.steps[pages.clamp(0, 8)][..., None, None]
    want[4:6] = 0
    assert torch.equal(bounds.values(pages), want) and bounds.values(pages[:0]).shape == (0, 3, 2, 128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = bounds.values(pages)
    side.synchronize()
    assert torch.equal(got, want)
    with pytest.raises(s3b.S3BError):
        bounds.values(pages.int())
    out, L = torch.empty(7, 3, 2, 128, device="cuda"), engine._L
    assert L.s3b_kv_bounds_values(bounds.ref, pages.data_ptr() + 4, 1, out.data_ptr(), None) == -1
    assert L.s3b_kv_bounds_values(bounds.ref, pages.data_ptr(), 1, out.data_ptr() + 4, None) == -1
    assert L.s3b_kv_bounds_values(bounds.ref, pages.data_ptr(), -1, out.data_ptr(), None) == -1
    assert L.s3b_kv_bounds_values(bounds.ref, None, 1, out.data_ptr(), None) == -1 and L.s3b_kv_bounds_values(None, None, 0, None, None) == -1


@pytest.mark.parametrize("new", [1, 2, 16, 17, 33, 500, 0])
def test_bounds_of_the_newest_tokens(s3b, engine, new):
    """Only the pages that hold the last `new` tokens are written, each over all of its tokens."""
    lengths, page = [97, 16, 1, 0, 130], 16
    q = Sequences(s3b, engine, 2, 64, 2, page, lengths, seed=new)
    every, some = s3b.KVBounds(q.cache), s3b.KVBounds(q.cache)
    engine.cache_bounds(q.cache, every, q.pages, q.lengths)
    some.codes.fill_(3)
    engine.cache_bounds(q.cache, some, q.pages, q.lengths, new=new)
    engine.sync()
    touched = torch.zeros(q.cache.n_pages, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lengths):
        if new:
            touched[q.pages[b, max(0, n - new) // page:-(-n // page)].long()] = True
    assert torch.equal(some.codes[touched], every.codes[touched]) and (some.codes[~touched] == 3).all()


@pytest.mark.parametrize("qtype", TYPES)
def test_bounds_of_odd_values(s3b, engine, qtype):
    """Pages of zeros, of one value, of f16's largest and least magnitudes."""
    cache = s3b.KVCache(qtype, 6, 16, 1, 64)
    x = torch.zeros(96, 1, 64, device="cuda")
    x[16:32] = -2.5
    x[32:48] = 65024.0
    x[48:64, :, ::2] = -65024.0
    x[64:80] = 6e-8
    x[80:96] = torch.linspace(-1e-6, 1e-6, 64, device="cuda")
    engine.cache_write(cache, x, x, torch.arange(96, device="cuda"))
    bounds = s3b.KVBounds(cache)
    engine.cache_bounds(cache, bounds, torch.arange(6, dtype=torch.int32, device="cuda")[None], torch.tensor([96], dtype=torch.int32, device="cuda"))
    k, v = (torch.empty(96, 1, 64, device="cuda", dtype=torch.float16) for _ in "kv")
    engine.cache_read(cache, torch.arange(96, device="cuda"), k, v)
    engine.sync()
    codes, steps = plain_bounds(k, 16)
    assert torch.equal(bounds.codes, codes) and torch.equal(bounds.steps, steps)


# ---------------------------------------------------------------- choice
def plain_scores(q, codes, steps):
    """Scores f32 [rows, pages] of query rows f16 [rows, d] by codes [pages, 2, d] and steps [pages]."""
    x = torch.nan_to_num(q.double(), nan=0.0, posinf=65504.0, neginf=-65504.0)
    peak = x.abs().amax(1, keepdim=True)
    inv = torch.where(peak > 0, 127 / peak, 0.0).float().double()
    c = (x * inv).float().round().clamp(-127, 127).double()
    dot = c.clamp(min=0) @ codes[:, 1].double().T + c.clamp(max=0) @ codes[:, 0].double().T
    return ((dot * steps.double()).float().double() * (peak / 127).float().double()).float()


def plain_choice(score, keep, sink, recent):
    """Places of the chosen of score [pages], a list."""
    n = len(score)
    if n <= keep:
        return list(range(n))
    order = sorted(range(sink, n - recent), key=lambda j: (-score[j], j))[:keep - sink - recent]
    return sorted([*range(sink), *order, *range(n - recent, n)])


def check_select(s3b, engine, s, q, keep, share, sink, recent, causal, window, bounds=None, want_scores=True):
    """Chooses with and without scores; compares both with the plain choice. Returns the lists."""
    batch, nq, heads, _ = q.shape
    group, page = heads // s.heads, s.page
    blocks = -(-nq // share)
    if bounds is None:
        bounds = s3b.KVBounds(s.cache)
        engine.cache_bounds(s.cache, bounds, s.pages, s.lengths)
    selected, again = (torch.full((batch, blocks, s.heads, keep), 9, dtype=torch.int32, device="cuda") for _ in "ab")
    scores = torch.full((batch, blocks, s.heads, s.pages.shape[1]), 5.0, device="cuda")
    args = dict(share=share, sink=sink, recent=recent, causal=causal, window=window)
    engine.cache_select(bounds, q, selected, s.pages, s.lengths, scores=scores, **args)
    engine.cache_select(bounds, q, again, s.pages, s.lengths, **args)
    engine.sync()
    assert torch.equal(selected, again)
    for b, n in enumerate(s.lens):
        sp = spans(n, nq, causal, window)
        for h in range(s.heads):
            at = s.pages[b].long()
            each = plain_scores(q[b, :, h * group:(h + 1) * group].reshape(-1, s.d), bounds.codes[at, h], bounds.steps[at, h]).view(nq, group, -1)
            for i in range(blocks):
                i0, i1 = i * share, min(nq, (i + 1) * share)
                lo, hi = sp[i0][0], sp[i1 - 1][1]
                pa = lo // page
                pe = max(pa, -(-hi // page))
                best = each[i0:i1].amax((0, 1))[pa:pe]
                want = torch.full((s.pages.shape[1],), -math.inf, device="cuda")
                want[pa:pe] = best
                assert torch.equal(scores[b, i, h], want), (b, h, i)
                chosen = [pa + j for j in plain_choice(best.tolist(), keep, sink, recent)]
                assert selected[b, i, h].tolist() == chosen + [-1] * (keep - len(chosen)), (b, h, i)
    return selected


@pytest.mark.parametrize("d,heads,kv,nq,share", [(64, 1, 1, 1, 1), (128, 8, 2, 1, 1), (256, 3, 1, 7, 5), (64, 10, 2, 6, 4), (128, 8, 1, 9, 4),
                                                 (256, 16, 1, 2, 1), (128, 6, 6, 3, 2), (64, 32, 1, 1, 1)])
@pytest.mark.parametrize("causal,window", [(False, 0), (True, 0), (True, 90)])
def test_select(s3b, engine, d, heads, kv, nq, share, causal, window):
    s = Sequences(s3b, engine, 8, d, kv, 16, [500, 0, 37, 3, 160], seed=d + heads)
    check_select(s3b, engine, s, s.queries(nq, heads), 5, share, 1, 2, causal, window)


@pytest.mark.parametrize("page,length,keep,sink,recent", [(16, 16 * 515, 40, 0, 0), (16, 8209, 8, 3, 5), (16, 65600, 100, 1, 1), (16, 70001, 1, 0, 0),
                                                          (16, 70001, 1, 1, 0), (32, 16384, 511, 0, 3), (16, 9000, 600, 300, 299)])
def test_select_of_many_pages(s3b, engine, page, length, keep, sink, recent):
    """Several blocks a list, more pages than a block keeps in registers, lists of one and of nearly all."""
    s = Sequences(s3b, engine, 2, 64, 2, page, [length, length // 3], seed=length)
    check_select(s3b, engine, s, s.queries(2, 4), keep, 2, sink, recent, True, 0)


@pytest.mark.parametrize("d,heads,kv,nq,share", [(64, 2, 2, 151, 1), (128, 16, 2, 300, 2), (256, 4, 1, 601, 2), (64, 4, 1, 1201, 4), (64, 4, 1, 2400, 8)])
@pytest.mark.parametrize("pages", [1, 40, 64, 65, 128, 129, 256, 257])
def test_select_of_many_lists(s3b, engine, d, heads, kv, nq, share, pages):
    """More lists than four an SM, whose blocks are as small as their pages allow; some of them of equal pages."""
    s = Sequences(s3b, engine, 2, d, kv, 16, [16 * pages - 3, 8 * pages], seed=pages + d)
    bounds = s3b.KVBounds(s.cache)
    engine.cache_bounds(s.cache, bounds, s.pages, s.lengths)
    engine.sync()
    bounds.codes[::3] = bounds.codes[0]
    bounds.steps[::3] = bounds.steps[0]
    check_select(s3b, engine, s, s.queries(nq, heads), 1 + pages // 3, share, min(1, pages // 3), 0, True, 0, bounds)


def test_select_ties(s3b, engine):
    """Equal pages: the lower ones; a query of zeros scores all pages 0."""
    s = Sequences(s3b, engine, 2, 64, 1, 16, [16 * 900], seed=5)
    bounds = s3b.KVBounds(s.cache)
    engine.cache_bounds(s.cache, bounds, s.pages, s.lengths)
    engine.sync()
    g = torch.Generator(device="cuda").manual_seed(1)
    same = torch.randint(0, 3, (s.cache.n_pages,), device="cuda", generator=g)  # three kinds of pages
    bounds.codes.copy_(bounds.codes[:3][same])
    bounds.steps.copy_(bounds.steps[:3][same])
    q = s.queries(3, 1)
    q[0, 1] = 0
    for keep, sink, recent in ((7, 0, 0), (400, 2, 3), (899, 0, 1)):
        check_select(s3b, engine, s, q, keep, 1, sink, recent, False, 0, bounds)


def test_select_of_odd_queries(s3b, engine):
    """NaN counts as 0, infinities as the largest; tiny and huge queries."""
    s = Sequences(s3b, engine, 8, 128, 1, 16, [700], seed=6)
    q = s.queries(6, 1)
    q[0, 0, 0, 5], q[0, 0, 0, 6] = math.nan, -math.nan
    q[0, 1, 0, 9], q[0, 2, 0, 100] = math.inf, -math.inf
    q[0, 3] = math.nan
    q[0, 4] *= 1e-6
    q[0, 5] = 65504.0
    check_select(s3b, engine, s, q, 4, 1, 0, 1, False, 0)


# ---------------------------------------------------------------- attention over chosen pages
def plain_attention(s, q, token, b, h, i0, i1, causal, window, scale, factor=1):
    """Output and ln sum exp of queries i0 .. i1 of one head group over the tokens (a tensor of positions), and bounds of their
    errors, in 64 bits."""
    batch, nq, heads, d = q.shape
    group = heads // s.heads
    k, v = (x[:, h].double() for x in s.rows(b))
    blocks = v.view(-1, d // 32, 32)
    size = (blocks.abs().amax(-1) + 2 * (blocks.amax(-1) - blocks.amin(-1))).repeat_interleave(32, -1) if s.cache.qtype == 3 else 0
    x = q[b, i0:i1, h * group:(h + 1) * group].reshape(-1, d).double()
    sp = torch.tensor(spans(len(k), nq, causal, window)[i0:i1], device="cuda").repeat_interleave(group, 0)
    e = (d + 16) * 2.0 ** -24 * scale * (x.abs() @ k[token].abs().T)
    z = (x @ k[token].T) * scale
    hide = (token < sp[:, :1]) | (token >= sp[:, 1:])
    z, e = z.masked_fill(hide, -math.inf), e.masked_fill(hide, 0.0).amax(1, keepdim=True) if len(token) else z.new_zeros(len(x), 1)
    p = z.softmax(-1).nan_to_num(0.0) if len(token) else z
    out = p @ v[token]
    err = (2 * torch.expm1(e) + U + 2.0 ** -19) * (p @ (v[token].abs() + (size[token] if s.cache.qtype == 3 else 0)))
    err += 2.0 ** -25 * len(token) * (v[token].abs().max() if len(token) else 0) + 1e-30
    lse = z.logsumexp(-1) if len(token) else torch.full((len(x),), -math.inf, device="cuda", dtype=torch.float64)
    lse_err = e[:, 0] + 2.0 ** -18 + (len(token) / 8 + 64) * 2.0 ** -24 + lse.abs().nan_to_num(posinf=0) * 2.0 ** -22
    return out, err, lse, lse_err


def check_attention(s3b, engine, s, q, selected, share, causal=False, window=0, out_type=torch.float16, strided=False):
    batch, nq, heads, d = q.shape
    group = heads // s.heads
    if strided:
        q = torch.cat([q, q], -1)[..., :d]
        out = torch.full((nq, batch, heads + 1, d + 16), 9.0, device="cuda", dtype=out_type)[:, :, 1:, 8:d + 8].transpose(0, 1)
    else:
        out = torch.full(q.shape, 9.0, device="cuda", dtype=out_type)
    lse, scale = torch.full(q.shape[:3], 9.0, device="cuda"), 0.9 * d ** -0.5
    engine.cache_attention_selected(s.cache, q, out, selected, s.pages, s.lengths, scale, share=share, causal=causal, window=window, lse=lse)
    again = torch.empty_like(out)
    engine.cache_attention_selected(s.cache, q, again, selected, s.pages, s.lengths, scale, share=share, causal=causal, window=window)
    engine.sync()
    assert torch.equal(out, again)
    for b, n in enumerate(s.lens):
        for i in range(selected.shape[1]):
            i0, i1 = i * share, min(nq, (i + 1) * share)
            for h in range(s.heads):
                names = selected[b, i, h].tolist()
                names = names[:next((x for x, y in enumerate(names) if y < 0), len(names))]
                token = torch.tensor([t for j in names for t in range(j * s.page, min(n, (j + 1) * s.page))], dtype=torch.int64, device="cuda")
                want, err, want_lse, lse_err = plain_attention(s, q, token, b, h, i0, i1, causal, window, scale)
                got = out[b, i0:i1, h * group:(h + 1) * group].reshape(-1, d).double()
                # a rounding of the output's type on top
                err = err + (U if out_type == torch.float16 else 2.0 ** -23) * want.abs() + (2.0 ** -25 if out_type == torch.float16 else 0)
                assert ((got - want).abs() <= err).all(), (b, i, h, ((got - want).abs() / err).max())
                got = lse[b, i0:i1, h * group:(h + 1) * group].reshape(-1).double()
                none = want_lse == -math.inf
                assert torch.equal(got == -math.inf, none), (b, i, h)
                assert ((got - want_lse).abs()[~none] <= lse_err[~none]).all(), (b, i, h)
    return out, lse


def lists(s, blocks, keep, g, order="ascending", holes=False):
    """Random lists of pages for every block and head."""
    out = torch.full((len(s.lens), blocks, s.heads, keep), -1, dtype=torch.int32)
    for b, n in enumerate(s.lens):
        pages = -(-n // s.page)
        for i in range(blocks):
            for h in range(s.heads):
                m = min(keep, pages)
                if holes and m:
                    m = int(torch.randint(0, m + 1, (), generator=g))
                names = torch.randperm(pages, generator=g)[:m].to(torch.int32)
                out[b, i, h, :m] = names.sort().values if order == "ascending" else names
    return out.cuda()


@pytest.mark.parametrize("qtype", TYPES)
@pytest.mark.parametrize("d,heads,kv,nq,share", [(64, 2, 2, 1, 1), (64, 12, 1, 4, 1), (64, 4, 1, 9, 8), (128, 8, 2, 3, 1), (128, 4, 1, 7, 3),
                                                 (128, 16, 1, 5, 2), (256, 1, 1, 20, 16), (256, 8, 1, 2, 1), (256, 3, 1, 5, 4)])
@pytest.mark.parametrize("page,lengths,keep", [(16, [130, 0, 16, 700], 6), (48, [49, 333], 3), (256, [600], 2)])
def test_attention_selected(s3b, engine, qtype, d, heads, kv, nq, share, page, lengths, keep):
    s = Sequences(s3b, engine, qtype, d, kv, page, lengths, seed=d + nq + page)
    g = torch.Generator().manual_seed(nq)
    check_attention(s3b, engine, s, s.queries(nq, heads), lists(s, -(-nq // share), keep, g), share)


@pytest.mark.parametrize("qtype", TYPES)
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 50), (True, 17)])
@pytest.mark.parametrize("out_type,strided", [(torch.float16, True), (torch.float32, False)])
def test_attention_selected_masks(s3b, engine, qtype, causal, window, out_type, strided):
    """Rows that see part of their pages or none of them, lists in any order that end early, sequences shorter than the queries."""
    s = Sequences(s3b, engine, qtype, 128, 2, 16, [200, 5, 0, 64, 1], seed=window)
    g = torch.Generator().manual_seed(window)
    check_attention(s3b, engine, s, s.queries(12, 4), lists(s, 3, 5, g, "any", holes=True), 4, causal, window, out_type, strided)


@pytest.mark.parametrize("qtype", TYPES)
@pytest.mark.parametrize("d,page,keep,heads", [(64, 16, 301, 2), (128, 16, 130, 8), (128, 64, 32, 4), (256, 32, 64, 16), (64, 48, 70, 32)])
def test_attention_selected_split(s3b, engine, qtype, d, page, keep, heads):
    """One list that many blocks share, its parts joined."""
    s = Sequences(s3b, engine, qtype, d, 1, page, [page * keep * 2 - 7], seed=page)
    g = torch.Generator().manual_seed(d)
    check_attention(s3b, engine, s, s.queries(1, heads), lists(s, 1, keep, g), 1)


@pytest.mark.parametrize("qtype,d", [(2, 128), (3, 256), (8, 64)])
def test_attention_selected_of_all_pages_is_attention(s3b, engine, qtype, d):
    s = Sequences(s3b, engine, qtype, d, 2, 32, [1000, 31, 400], seed=3)
    q = s.queries(5, 4)
    every = torch.arange(s.pages.shape[1], dtype=torch.int32, device="cuda").expand(3, 5, 2, -1).contiguous()
    out, lse = check_attention(s3b, engine, s, q, torch.where(every * 32 < s.lengths[:, None, None, None], every, -1), 1, True, 300, torch.float32)
    dense, dense_lse = torch.empty_like(out), torch.empty_like(lse)
    engine.cache_attention(s.cache, q, dense, s.pages, s.lengths, 0.9 * d ** -0.5, causal=True, window=300, lse=dense_lse)
    engine.sync()
    assert (out - dense).norm() <= 4 * U * dense.norm()  # cache_attention rounds a weight twice
    assert torch.equal(lse == -math.inf, dense_lse == -math.inf)
    seen = lse > -math.inf
    assert (lse - dense_lse)[seen].abs().max() < 2.0 ** -14


def test_attention_selected_behind_the_sequence(s3b, engine):
    """Entries past the last page of the sequence but inside the table see nothing, whatever the table holds there."""
    s = Sequences(s3b, engine, 2, 64, 1, 16, [40, 100], seed=8)
    s.pages[0, 3:] = -5
    selected = torch.tensor([[[[0, 5, 2, 6]]], [[[6, 1, -1, 0]]]], dtype=torch.int32, device="cuda")
    check_attention(s3b, engine, s, s.queries(1, 1), selected, 1)


@pytest.mark.parametrize("qtype,d,page", [(2, 64, 16), (3, 128, 16), (8, 256, 32)])
def test_attention_selected_by_any_list(s3b, engine, qtype, d, page):
    """Pages named twice count twice; pages behind the sequence, first in the list, take no page's place; lists longer than the
    sequence, in one block and cut into parts."""
    s = Sequences(s3b, engine, qtype, d, 1, page, [3 * page - 5, 40 * page], seed=d, width=60)
    g = torch.Generator().manual_seed(d)
    for keep in (7, 200):
        selected = torch.randint(0, 60, (2, 2, 1, keep), generator=g, dtype=torch.int32)
        selected[0, 0, 0, :4] = torch.tensor([50, 59, 2, 2])
        selected[0, 0, 0, 4:] = torch.randint(0, 3, (keep - 4,), generator=g, dtype=torch.int32)
        selected[1, 1, 0, keep - 2:] = -1
        check_attention(s3b, engine, s, s.queries(2, 2), selected.cuda(), 1)


@pytest.mark.parametrize("size", [1e-3, 1.0, 300.0])
@pytest.mark.parametrize("qtype", TYPES)
def test_attention_selected_of_values_of_any_size(s3b, engine, qtype, size):
    """One page far larger or smaller than the others, met late."""
    s = Sequences(s3b, engine, qtype, 64, 1, 16, [16 * 40], seed=9)
    k, v = s.rows(0)
    v[300:316] *= size
    engine.cache_write(s.cache, k, v, s.slots[0, :640].contiguous())
    g = torch.Generator().manual_seed(4)
    check_attention(s3b, engine, s, s.queries(2, 1), lists(s, 2, 30, g), 1, out_type=torch.float32)


# ---------------------------------------------------------------- gathered weights
def check_weights(engine, s, q, causal=False, window=0, decay=1.0, weights=None, lse=None):
    batch, nq, heads, d = q.shape
    group, tokens, scale = heads // s.heads, s.pages.shape[1] * s.page, 0.9 * d ** -0.5
    if weights is None:
        weights = torch.rand(batch, s.heads, tokens, device="cuda", generator=s.g)
    before = weights.double().clone()
    sums, held = [], [s.rows(b)[0].double() for b in range(batch)]
    if lse is None:
        lse = torch.full((batch, nq, heads), -math.inf, device="cuda")
        for b, n in enumerate(s.lens):
            sp = torch.tensor(spans(n, nq, causal, window), device="cuda")
            at = torch.arange(n, device="cuda")
            for h in range(heads):
                z = q[b, :, h].double() @ held[b][:, h // group].T * scale
                if n:
                    lse[b, :, h] = z.masked_fill((at < sp[:, :1]) | (at >= sp[:, 1:]), -math.inf).logsumexp(-1).float()
    engine.cache_weights(s.cache, q, lse, weights, s.pages, s.lengths, scale, decay=decay, causal=causal, window=window)
    engine.sync()
    for b, n in enumerate(s.lens):
        sp = torch.tensor(spans(n, nq, causal, window), device="cuda").view(nq, 2)
        at = torch.arange(n, device="cuda")
        for h in range(s.heads):
            want, err = decay * before[b, h, :n], torch.zeros(n, device="cuda", dtype=torch.float64)
            for m in range(h * group, (h + 1) * group):
                x, k = q[b, :, m].double(), held[b][:, h]
                z, r = x @ k.T * scale, lse[b, :, m, None].double()
                hide = (at < sp[:, :1]) | (at >= sp[:, 1:]) | (r == -math.inf)
                p = torch.exp(z - r).masked_fill(hide, 0.0)
                # the score's error, that of its product with log2 e and of the difference, ex2's
                e = (d + 16) * 2.0 ** -24 * scale * (x.abs() @ k.abs().T) + (z.abs() + 2 * r.abs()) * 2.0 ** -23 + 2.0 ** -21
                err += (p * torch.expm1(e)).nan_to_num(0.0).sum(0)
                want = want + p.sum(0)
            err += (nq * group + 4) * 2.0 ** -24 * want + 1e-30
            got = weights[b, h, :n].double()
            assert ((got - want).abs() <= err).all(), (b, h, ((got - want).abs() / err).max())
            sums.append((got - decay * before[b, h, :n]).sum().item())
            assert torch.equal(weights[b, h, n:].double(), before[b, h, n:])
    return sums


@pytest.mark.parametrize("qtype", TYPES)
@pytest.mark.parametrize("d,heads,kv,nq", [(64, 1, 1, 1), (64, 12, 4, 5), (128, 8, 2, 1), (128, 4, 1, 33), (256, 1, 1, 130), (256, 6, 2, 3), (128, 3, 3, 40)])
@pytest.mark.parametrize("page,lengths", [(16, [1, 300, 0]), (48, [577]), (80, [100, 640, 79, 81])])
def test_weights(s3b, engine, qtype, d, heads, kv, nq, page, lengths):
    s = Sequences(s3b, engine, qtype, d, kv, page, lengths, seed=nq + page)
    sums = check_weights(engine, s, s.queries(nq, heads), decay=0.9)
    for total, n in zip(sums, [n for n in lengths for _ in range(kv)]):  # every row gives 1 in all
        assert abs(total - (nq * heads // kv if n else 0)) <= 1e-3 * nq * heads


@pytest.mark.parametrize("qtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("heads,kv,nq,lengths", [(1, 1, 129, [1]), (3, 1, 100, [130, 0, 1000]), (2, 2, 513, [129, 128, 127]), (8, 1, 64, [3000]), (4, 2, 700, [5000, 17])])
@pytest.mark.parametrize("causal,window", [(False, 0), (True, 0), (True, 200)])
def test_weights_of_many_rows(s3b, engine, qtype, d, heads, kv, nq, lengths, causal, window):
    """Tiles of 128 tokens and 128 rows: one tile, heads that fill no tile, tiles that several blocks share, long walks."""
    s = Sequences(s3b, engine, qtype, d, kv, 48, lengths, seed=nq + d)
    check_weights(engine, s, s.queries(nq, heads), causal, window, 0.5)


@pytest.mark.parametrize("qtype,d", [(2, 64), (3, 128), (8, 256)])
@pytest.mark.parametrize("window", [0, 9, 100])
@pytest.mark.parametrize("nq", [1, 7, 200])
def test_weights_masks(s3b, engine, qtype, d, window, nq):
    s = Sequences(s3b, engine, qtype, d, 2, 16, [250, 3, 0, 100], seed=window)
    check_weights(engine, s, s.queries(nq, 4), True, window, 1.0)


def test_weights_of_rows_that_saw_nothing(s3b, engine):
    """A row with -inf adds nothing, also where the call's mask shows it tokens; NaN queries of such rows stay out."""
    s = Sequences(s3b, engine, 2, 64, 1, 16, [100], seed=2)
    q = s.queries(3, 2)
    q[0, 1] = math.nan
    lse = torch.full((1, 3, 2), 4.0, device="cuda")
    lse[0, 1] = -math.inf
    w = torch.zeros(1, 1, 112, device="cuda")
    v = torch.zeros(1, 1, 112, device="cuda")
    engine.cache_weights(s.cache, q, lse, w, s.pages, s.lengths, 0.1)
    engine.cache_weights(s.cache, q[:, ::2].contiguous(), lse[:, ::2].contiguous(), v, s.pages, s.lengths, 0.1)
    engine.sync()
    assert torch.isfinite(w).all() and (w - v).abs().max() <= 1e-6 * v.max() and w[0, 0, 99] > 0 and (w[0, 0, 100:] == 0).all()


@pytest.mark.parametrize("nq,heads", [(1, 2), (20, 2), (200, 2)])
def test_weights_with_a_decay_of_zero(s3b, engine, nq, heads):
    """What was there does not count, whatever it is; tokens that no row sees end at 0, those behind the last keep theirs."""
    s = Sequences(s3b, engine, 2, 64, 2, 16, [300, 17], seed=nq)
    w = torch.full((2, 2, 304), math.nan, device="cuda")
    v = torch.zeros(2, 2, 304, device="cuda")
    q, lse = s.queries(nq, heads), torch.full((2, nq, heads), 3.0, device="cuda")
    for x in (w, v):
        engine.cache_weights(s.cache, q, lse, x, s.pages, s.lengths, 0.1, decay=0.0, causal=True, window=5)
    engine.sync()
    for b, n in enumerate(s.lens):
        assert torch.equal(w[b, :, :n], v[b, :, :n]) and torch.isnan(w[b, :, n:]).all()
    assert (w[0, :, :300 - nq - 4] == 0).all() and (w[0, :, 299] > 0).all()


@pytest.mark.parametrize("nq", [1, 40, 300])
def test_wide_page_tables_cost_nothing(s3b, engine, nq):
    """Tables of 2^27 tokens with short sequences: the lengths say what is done."""
    s = Sequences(s3b, engine, 2, 128, 2, 64, [200, 0, 1000], seed=nq)
    wide = torch.zeros(1, 1 << 21, dtype=torch.int32, device="cuda")
    table = wide.expand(3, -1).clone()
    table[:, :s.pages.shape[1]] = s.pages
    q, lse = s.queries(nq, 4), torch.full((3, nq, 4), 3.0, device="cuda")
    w, v = torch.ones(3, 2, 64 << 21, device="cuda"), torch.ones(3, 2, 1024, device="cuda")
    engine.cache_weights(s.cache, q, lse, w, table, s.lengths, 0.1, causal=True)
    engine.cache_weights(s.cache, q, lse, v, s.pages, s.lengths, 0.1, causal=True)
    bounds, again = s3b.KVBounds(s.cache), s3b.KVBounds(s.cache)
    engine.cache_bounds(s.cache, bounds, table, s.lengths)
    engine.cache_bounds(s.cache, again, s.pages, s.lengths)
    a, b = (torch.empty(3, -(-nq // 8), 2, 4, dtype=torch.int32, device="cuda") for _ in "ab")
    engine.cache_select(bounds, q, a, table, s.lengths, share=8)
    engine.cache_select(bounds, q, b, s.pages, s.lengths, share=8)
    x, y = torch.empty_like(q), torch.empty_like(q)
    engine.cache_attention_selected(s.cache, q, x, a, table, s.lengths, 0.1, share=8)
    engine.cache_attention_selected(s.cache, q, y, b, s.pages, s.lengths, 0.1, share=8)
    engine.sync()
    assert torch.equal(w[:, :, :1024], v) and (w[:, :, 1024:] == 1).all()
    assert torch.equal(bounds.codes, again.codes) and torch.equal(a, b) and torch.equal(x, y)


@pytest.mark.parametrize("nq", [1, 70])
def test_weights_rows_apart(s3b, engine, nq):
    """Weights and queries as slices of larger tensors, sequences inside and heads outside."""
    s = Sequences(s3b, engine, 8, 128, 3, 16, [90, 33], seed=4)
    wide = torch.rand(3, 2, 200, device="cuda")
    kept = wide.clone()
    weights = wide[:, :, 7:7 + 96].transpose(0, 1)
    q = torch.cat([s.queries(nq, 6)] * 2, 1)[:, nq:]
    check_weights(engine, s, q, weights=weights, decay=0.0)
    assert torch.equal(wide[:, :, :7], kept[:, :, :7]) and torch.equal(wide[:, :, 103:], kept[:, :, 103:])


# ---------------------------------------------------------------- eviction
def check_evict(s3b, engine, s, weights, keep, sink=0, recent=0, to=None, extra=0):
    """Evicts into other pages of the cache (or into `to`) and compares positions, weights and rows bit for bit."""
    batch = len(s.lens)
    cache = s.cache
    target = cache if to is None else to
    new_pages = -(-max(keep, 1) // target.page_size) + extra
    if to is None:
        free = torch.ones(cache.n_pages, dtype=torch.bool, device="cuda")
        free[s.pages.long().flatten()] = False
        pages_out = free.nonzero()[:batch * new_pages, 0].to(torch.int32).view(batch, new_pages)
    else:
        pages_out = torch.arange(batch * new_pages, device="cuda").flip(0).to(torch.int32).view(batch, new_pages)
    lengths_out = torch.full((batch,), -3, dtype=torch.int32, device="cuda")
    kept = torch.full((batch, s.heads, keep), 9, dtype=torch.int32, device="cuda")
    weights_out = torch.full((batch, s.heads, keep), 9.0, device="cuda")
    before = cache.data.clone()
    target_before = target.data.clone()
    rows = [s.rows(b) for b in range(batch)]
    engine.cache_evict(cache, weights, s.pages, s.lengths, pages_out, lengths_out, kept, sink=sink, recent=recent, weights_out=weights_out, to=to)
    engine.sync()
    assert lengths_out.tolist() == [min(n, keep) for n in s.lens]
    slots = (pages_out.long()[:, :, None] * target.page_size + torch.arange(target.page_size, device="cuda")).flatten(1)
    for b, n in enumerate(s.lens):
        m = min(n, keep)
        k, v = (torch.empty(m, s.heads, s.d, device="cuda") for _ in "kv")
        engine.cache_read(target, slots[b, :m].contiguous(), k, v)
        engine.sync()
        for h in range(s.heads):
            w = weights[b, h, :n].tolist()
            w = [-math.inf if x != x else x for x in w]
            rank = [(0 if x == x else 1) for x in weights[b, h, :n].tolist()]
            if n <= keep:
                chosen = list(range(n))
            else:
                order = sorted(range(sink, n - recent), key=lambda j: (rank[j], -w[j], j))[:keep - sink - recent]
                chosen = sorted([*range(sink), *order, *range(n - recent, n)])
            assert kept[b, h].tolist() == chosen + [-1] * (keep - m), (b, h)
            at = torch.tensor(chosen, dtype=torch.int64, device="cuda")
            assert torch.equal(weights_out[b, h, :m].view(torch.int32), weights[b, h, at].view(torch.int32)) and (weights_out[b, h, m:] == 0).all()
            assert torch.equal(k[:, h], rows[b][0][at, h]) and torch.equal(v[:, h], rows[b][1][at, h]), (b, h)
    # what the call does not write: the source, other pages, places behind the last
    if to is not None:
        assert torch.equal(cache.data, before)
    if (1 << 22) > target.n_slots * s.heads * s.d:
        other = torch.ones(target.n_slots, dtype=torch.bool, device="cuda")
        for b, n in enumerate(s.lens):
            other[slots[b, :min(n, keep)]] = False
        other = other.nonzero()[:, 0].contiguous()
        now, then = ([torch.empty(len(other), s.heads, s.d, device="cuda") for _ in "kv"] for _ in "ab")
        engine.cache_read(target, other, *now)
        engine.cache_read(s3b.KVCache(target.qtype, target.n_pages, target.page_size, s.heads, s.d, data=target_before), other, *then)
        engine.sync()
        assert torch.equal(now[0], then[0]) and torch.equal(now[1], then[1])
    return kept


def some_weights(s, ties=False):
    w = torch.exp(2 * torch.randn(len(s.lens), s.heads, s.pages.shape[1] * s.page, device="cuda", generator=s.g))
    return torch.where(torch.rand(w.shape, device="cuda", generator=s.g) < 0.3, 0.0, w.round() if ties else w)


@pytest.mark.parametrize("qtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page,heads,lengths,keep,sink,recent", [(16, 1, [40], 16, 0, 0), (48, 3, [200, 0, 97, 30], 37, 2, 9), (32, 2, [333, 65], 64, 60, 4),
                                                                 (16, 2, [33], 1, 0, 0)])
def test_evict(s3b, engine, qtype, d, page, heads, lengths, keep, sink, recent):
    s = Sequences(s3b, engine, qtype, d, heads, page, lengths, seed=d, spare=len(lengths) * 5)
    check_evict(s3b, engine, s, some_weights(s, ties=True), keep, sink, recent)


@pytest.mark.parametrize("qtype", TYPES)
def test_evict_into_another_cache(s3b, engine, qtype):
    s = Sequences(s3b, engine, qtype, 128, 2, 64, [300, 129], seed=1)
    check_evict(s3b, engine, s, some_weights(s), 100, 3, 3, to=s3b.KVCache(qtype, 20, 16, 2, 128), extra=1)


@pytest.mark.parametrize("length,keep,heads", [(16384, 5000, 1), (16385, 16384, 2), (40000, 77, 1), (140001, 3000, 1), (200003, 150000, 2)])
@pytest.mark.parametrize("ties", [False, True])
def test_evict_long(s3b, engine, length, keep, heads, ties):
    """Up to and past what one block, and eight, keep in registers."""
    s = Sequences(s3b, engine, 2, 64, heads, 16, [length, length // 2], seed=length, spare=2 * (keep // 16 + 1))
    check_evict(s3b, engine, s, some_weights(s, ties), keep, 4, 100 if keep > 104 else 0)


def test_evict_odd_weights(s3b, engine):
    """Infinities, NaN below all, zeros of both signs equal, negative weights, all equal."""
    s = Sequences(s3b, engine, 2, 64, 6, 16, [100], seed=3, spare=8)
    w = some_weights(s)
    w[0, 0, ::3], w[0, 0, 1::7] = math.inf, -math.inf
    w[0, 1, ::2], w[0, 1, 5] = math.nan, -math.nan
    w[0, 2] = 0.0
    w[0, 2, ::2] = -0.0
    w[0, 3] = -torch.arange(112, device="cuda").float()
    w[0, 4] = 1.5
    w[0, 5] = math.nan
    for keep, sink, recent in ((30, 0, 0), (30, 5, 5), (99, 1, 1), (100, 0, 0), (112, 50, 62)):
        check_evict(s3b, engine, s, w, keep, sink, recent)


def test_evict_nothing_kept(s3b, engine):
    s = Sequences(s3b, engine, 2, 64, 1, 16, [50, 3], seed=3)
    lengths_out = torch.full((2,), 5, dtype=torch.int32, device="cuda")
    engine.cache_evict(s.cache, some_weights(s), s.pages, s.lengths, torch.empty(2, 0, dtype=torch.int32, device="cuda"), lengths_out,
                       torch.empty(2, 1, 0, dtype=torch.int32, device="cuda"))
    engine.sync()
    assert lengths_out.tolist() == [0, 0]


@pytest.mark.parametrize("qtype,d", [(2, 64), (3, 128), (8, 256), (2, 256)])
@pytest.mark.parametrize("nq", [1, 40, 300])
def test_memory_that_was_never_written(s3b, engine, qtype, d, nq):
    """A cache in memory of all ones (scales of NaN) gives the same bits as one in zeros, wherever no token lies; so do the places that
    an eviction into such a cache leaves."""
    heads, page, n, most, keep = 2, 48, 437, 12, 100
    pages, lengths = torch.arange(most, dtype=torch.int32, device="cuda")[None], torch.tensor([n], dtype=torch.int32, device="cuda")
    results = []
    for fill in (0, 255):
        g = torch.Generator(device="cuda").manual_seed(d + nq)
        c, to = (s3b.KVCache(qtype, most, page, heads, d, data=torch.full((s3b.kv_cache_bytes(qtype, heads, d, page, most),), fill, dtype=torch.uint8, device="cuda"))
                 for _ in "ab")
        k, v = (torch.randn(n, heads, d, device="cuda", generator=g).half() for _ in "kv")
        engine.cache_write(c, k, v, torch.arange(n, device="cuda"))
        q, bounds = torch.randn(1, nq, heads, d, device="cuda", generator=g).half(), s3b.KVBounds(c)
        out, dense, again = torch.empty_like(q), torch.empty_like(q), torch.empty_like(q)
        lse, weights = torch.empty(1, nq, heads, device="cuda"), torch.zeros(1, heads, most * page, device="cuda")
        selected, scores = torch.empty(1, nq, heads, 6, dtype=torch.int32, device="cuda"), torch.empty(1, nq, heads, most, device="cuda")
        kept, length = torch.empty(1, heads, keep, dtype=torch.int32, device="cuda"), torch.empty(1, dtype=torch.int32, device="cuda")
        engine.cache_attention(c, q, dense, pages, lengths, d ** -0.5, lse=lse)
        engine.cache_bounds(c, bounds, pages, lengths)
        engine.cache_select(bounds, q, selected, pages, lengths, scores=scores)
        engine.cache_attention_selected(c, q, out, selected, pages, lengths, d ** -0.5)
        engine.cache_weights(c, q, lse, weights, pages, lengths, d ** -0.5)
        engine.cache_evict(c, weights, pages, lengths, pages, length, kept, to=to)
        engine.cache_attention(to, q, again, pages, length, d ** -0.5)
        engine.sync()
        assert all(torch.isfinite(x).all() for x in (out, weights, again))
        results.append((out, lse, weights, selected, scores, bounds.codes, bounds.steps, kept, again))
    assert all(torch.equal(x, y) for x, y in zip(*results))
