"""Long caches at the edges of what the calls take. Plain forms, tolerances and inputs as in test_kv_long_gpu.py."""
import math

import pytest

torch = pytest.importorskip("torch")
from test_kv_long_gpu import Sequences, check_evict, plain_attention, plain_choice, plain_scores, some_weights  # noqa: E402
from test_kv_long_run_gpu import raw  # noqa: E402, F401

pytestmark = pytest.mark.gpu


def needs(gigabytes):
    if torch.cuda.mem_get_info()[0] < gigabytes * 2 ** 30:
        pytest.skip(f"needs {gigabytes} GB of device memory")


# ---------------------------------------------------------------- empty sequences
def test_an_empty_sequence_of_2_to_the_25_queries(s3b, engine):
    """More than 2^31 pieces of four outputs: all rows are zero, all ln sums -inf."""
    needs(22)
    nq, d, share = 2 ** 25 + 3, 256, 16
    cache = s3b.KVCache(2, 1, 16, 1, d)
    q = torch.ones(1, 1, 1, d, dtype=torch.float16, device="cuda").expand(1, nq, 1, d)
    out, lse = torch.full((1, nq, 1, d), 9.0, dtype=torch.float16, device="cuda"), torch.full((1, nq, 1), 9.0, device="cuda")
    selected = torch.zeros(1, -(-nq // share), 1, 1, dtype=torch.int32, device="cuda")
    engine.cache_attention_selected(cache, q, out, selected, torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                                    torch.zeros(1, dtype=torch.int32, device="cuda"), 0.1, share=share, lse=lse)
    engine.sync()
    assert (lse == -math.inf).all()
    words = out.view(-1).view(torch.int64)
    for i in range(0, len(words), 2 ** 28):
        assert not words[i:i + 2 ** 28].any()
    del out, words
    torch.cuda.empty_cache()


@pytest.mark.parametrize("qtype,d,heads,kv,nq,share,lengths", [
    (2, 128, 32, 8, 2050, 4, [300, 0, 170]), (3, 64, 3, 1, 4099, 10, [0, 0, 65, 0]), (8, 256, 2, 2, 3001, 16, [64, 0]), (2, 64, 1, 1, 127, 1, [0, 5, 0]),
    (2, 64, 1, 1, 129, 1, [0, 0])])
@pytest.mark.parametrize("out_type", [torch.float16, torch.float32])
def test_empty_sequences_beside_others(s3b, engine, qtype, d, heads, kv, nq, share, lengths, out_type):
    """Rows of empty sequences are zero, those of the others as without them, and nothing between the rows is written."""
    s = Sequences(s3b, engine, qtype, d, kv, 16, lengths, seed=nq)
    q, scale = s.queries(nq, heads), d ** -0.5
    batch, blocks, keep = len(lengths), -(-nq // share), 3
    selected = torch.randint(0, 4, (batch, blocks, kv, keep), generator=torch.Generator().manual_seed(1), dtype=torch.int32).cuda()
    selected.clamp_(max=s.pages.shape[1] - 1)
    wide = torch.full((batch, nq, heads + 1, d + 16), 9.0, dtype=out_type, device="cuda")
    lse = torch.full((batch, nq, heads), 9.0, device="cuda")
    out = wide[:, :, :heads, 8:d + 8]
    engine.cache_attention_selected(s.cache, q, out, selected, s.pages, s.lengths, scale, share=share, lse=lse)
    engine.sync()
    for b, n in enumerate(lengths):
        if not n:
            assert (out[b] == 0).all() and (lse[b] == -math.inf).all()
            continue
        alone, alone_lse = torch.empty(1, nq, heads, d, dtype=out_type, device="cuda"), torch.empty(1, nq, heads, device="cuda")
        engine.cache_attention_selected(s.cache, q[b:b + 1], alone, selected[b:b + 1], s.pages[b:b + 1], s.lengths[b:b + 1], scale, share=share, lse=alone_lse)
        engine.sync()
        # blocks may share a unit in another way: f32 sums in another order, then the output's rounding
        assert (alone[0].double() - out[b].double()).norm() <= 2.0 ** -10 * alone[0].double().norm()
        assert (alone_lse[0] - lse[b]).abs().max() <= 2.0 ** -16
    assert (wide[:, :, heads] == 9).all() and (wide[..., :8] == 9).all() and (wide[..., d + 8:] == 9).all()


@pytest.mark.parametrize("nq,heads,lengths", [(1, 8, [0, 40, 0]), (7, 32, [0] * 5 + [100] + [0] * 300), (32, 4, [0])])
def test_empty_sequences_of_the_dense_attention(s3b, engine, nq, heads, lengths):
    """The same rows by the call over all pages, which shares the kernel."""
    s = Sequences(s3b, engine, 2, 64, 4, 16, lengths, seed=nq)
    q = s.queries(nq, heads)
    out, lse = torch.full(q.shape, 9.0, device="cuda"), torch.full(q.shape[:3], 9.0, device="cuda")
    engine.cache_attention(s.cache, q, out, s.pages, s.lengths, 0.1, lse=lse)
    engine.sync()
    none = s.lengths == 0
    assert (out[none] == 0).all() and (lse[none] == -math.inf).all()
    assert torch.isfinite(lse[~none]).all() and (out[~none] != 9).all()


# ---------------------------------------------------------------- positions near 2^31
def test_a_sequence_of_nearly_2_to_the_31_tokens(s3b, engine):
    """The last page's end, rounded up to whole pages, passes 2^31. All entries of the table name two pages in turn."""
    page, width = 8208, 261632
    length = page * width  # 2^31 - 8192, the longest that there is
    cache = s3b.KVCache(2, 2, page, 1, 64)
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(2 * page, 1, 64, device="cuda", generator=g).half() for _ in "kv")
    engine.cache_write(cache, k, v, torch.arange(2 * page, device="cuda"))
    pages = (torch.arange(width, dtype=torch.int32, device="cuda") % 2)[None]
    lengths = torch.tensor([length], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 2, 1, 64, device="cuda", generator=g).half()
    selected = torch.tensor([[0, width - 1, -1], [width - 1, width - 2, 7]], dtype=torch.int32, device="cuda")[None, :, None]
    out, lse = torch.full(q.shape, 9.0, device="cuda"), torch.full((1, 2, 1), 9.0, device="cuda")
    # with a window, query 0 sees the last 9000 tokens up to the one before the last
    for window in (0, 9000):
        engine.cache_attention_selected(cache, q, out, selected, pages, lengths, 0.125, causal=True, window=window, lse=lse)
        engine.sync()
        held = [torch.empty(2 * page, 1, 64, device="cuda") for _ in "kv"]
        engine.cache_read(cache, torch.arange(2 * page, device="cuda"), *held)
        engine.sync()
        for i in range(2):
            names = [x for x in selected[0, i, 0].tolist() if x >= 0]
            at = torch.cat([torch.arange(page, device="cuda") + x * page for x in names])
            hi = length - 1 + i
            seen = (at < hi) & (at >= (hi - window if window else 0))
            row = (at // page % 2 * page + at % page)[seen]
            z = held[0][row, 0].double() @ q[0, i, 0].double() * 0.125
            want = z.softmax(0) @ held[1][row, 0].double()
            assert (out[0, i, 0] - want).norm() <= 2.0 ** -10 * want.norm()  # at most two roundings to f16, of half a step each
            assert abs(lse[0, i, 0].item() - z.logsumexp(0).item()) <= 2.0 ** -16


# ---------------------------------------------------------------- how a choice holds its keys
class Bounded:
    """Sequences over one page table of `pages` pages, of which only random bounds are looked at."""

    def __init__(self, s3b, heads, d, pages, lengths, seed=0):
        self.heads, self.d, self.page, self.lens = heads, d, 16, lengths
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.cache = s3b.KVCache(2, pages, 16, heads, d)
        self.pages = torch.randperm(pages, device="cuda", generator=self.g).to(torch.int32).expand(len(lengths), -1)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        self.bounds = s3b.KVBounds(self.cache)
        low = torch.randint(-127, 128, (pages, heads, d), device="cuda", generator=self.g)
        high = torch.randint(-127, 128, (pages, heads, d), device="cuda", generator=self.g)
        self.bounds.codes[:, :, 0], self.bounds.codes[:, :, 1] = torch.minimum(low, high), torch.maximum(low, high)
        self.bounds.steps.copy_(torch.rand(pages, heads, device="cuda", generator=self.g))
        # a quarter of the pages are equal, so that the choice ends among equals
        self.bounds.codes[::4], self.bounds.steps[::4] = self.bounds.codes[0], self.bounds.steps[0]

    def queries(self, nq, heads):
        return torch.randn(len(self.lens), nq, heads, self.d, device="cuda", generator=self.g).half()


@pytest.mark.parametrize("batch,heads,pages,keep", [
    (160, 1, 600, 40), (32, 5, 700, 300), (160, 1, 24576, 100), (160, 1, 24577, 5000), (53, 3, 26000, 26),  # a block of 8 warps a list
    (40, 1, 1025, 33), (10, 4, 3000, 1500), (40, 1, 24576, 24000), (38, 1, 25001, 200),                      # 16 warps
    (20, 1, 50000, 64), (5, 1, 200000, 1000), (1, 2, 400000, 77)])                                           # clusters of 2, 8 and 16
def test_select_rounds(s3b, engine, batch, heads, pages, keep):
    """Lists whose threshold is found digit by digit, in one block and in clusters, with keys in shared memory and remade from the
    scores where more than 24576 pages fall to a block."""
    lengths = [16 * pages - (i % 5) * (pages // 7) * 16 - i % 16 for i in range(batch)]
    s = Bounded(s3b, heads, 64, pages, lengths, seed=pages)
    q = s.queries(1, heads)
    selected, again = (torch.full((batch, 1, heads, keep), 9, dtype=torch.int32, device="cuda") for _ in "ab")
    scores = torch.full((batch, 1, heads, pages), 5.0, device="cuda")
    engine.cache_select(s.bounds, q, selected, s.pages, s.lengths, sink=1, recent=2, scores=scores)
    engine.cache_select(s.bounds, q, again, s.pages, s.lengths, sink=1, recent=2)
    engine.sync()
    assert torch.equal(selected, again)
    some = range(batch) if pages < 2000 else sorted({0, batch // 3, batch - 1})
    at = s.pages[0].long()
    for b in some:
        n = -(-lengths[b] // 16)
        for h in range(heads):
            want = plain_scores(q[b, :, h], s.bounds.codes[at, h], s.bounds.steps[at, h])[0]
            assert torch.equal(scores[b, 0, h, :n], want[:n]) and (scores[b, 0, h, n:] == -math.inf).all()
            chosen = plain_choice(want[:n].tolist(), keep, 1, 2)
            assert selected[b, 0, h].tolist() == chosen + [-1] * (keep - len(chosen)), (b, h)


def test_select_of_many_lists_of_very_many_pages(s3b, engine):
    """Lists whose scores, kept at once, would take 270 MB: the same as a few at a time."""
    batch, pages, keep = 160, 430000, 50
    s = Bounded(s3b, 1, 64, pages, [16 * pages - 16 * 1000 * i for i in range(batch)], seed=3)
    q = s.queries(1, 1)
    selected, few = (torch.full((batch, 1, 1, keep), 9, dtype=torch.int32, device="cuda") for _ in "ab")
    engine.cache_select(s.bounds, q, selected, s.pages, s.lengths)
    for b in range(0, batch, 40):
        engine.cache_select(s.bounds, q[b:b + 40], few[b:b + 40], s.pages[b:b + 40], s.lengths[b:b + 40])
    engine.sync()
    assert torch.equal(selected, few)
    at = s.pages[0].long()
    for b in (0, 159):
        n = -(-s.lens[b] // 16)
        want = plain_scores(q[b, :, 0], s.bounds.codes[at, 0], s.bounds.steps[at, 0])[0, :n]
        assert selected[b, 0, 0].tolist() == plain_choice(want.tolist(), keep, 0, 1)


@pytest.mark.parametrize("width", [32769, 1 << 21])
def test_select_by_tables_far_wider_than_their_sequences(s3b, engine, width):
    """Some thousand lists over a table whose scores would not fit the GPU, or would fill much of it: the lists of a narrow table."""
    s = Sequences(s3b, engine, 2, 64, 4, 64, [1000, 3000], seed=4)
    table = torch.full((2, width), -7, dtype=torch.int32, device="cuda")
    table[:, :s.pages.shape[1]] = s.pages
    bounds = s3b.KVBounds(s.cache)
    engine.cache_bounds(s.cache, bounds, s.pages, s.lengths)
    q = s.queries(4096, 4)
    before = torch.cuda.mem_get_info()[0]
    wide, narrow = (torch.full((2, 4096, 4, 4), 9, dtype=torch.int32, device="cuda") for _ in "ab")
    engine.cache_select(bounds, q, wide, table, s.lengths, causal=True)
    engine.cache_select(bounds, q, narrow, s.pages, s.lengths, causal=True)
    engine.sync()
    assert torch.equal(wide, narrow)
    assert before - torch.cuda.mem_get_info()[0] <= 2 ** 29  # no workspace of all scores stays behind


# ---------------------------------------------------------------- how an eviction holds its keys
@pytest.mark.parametrize("lengths,heads,keep", [
    ([3000, 2049], 75, 1000), ([2500], 80, 2499), ([49152], 76, 300), ([50001], 75, 20000),  # a block a head: in shared memory, remade
    ([800003], 1, 3000), ([800003, 790000], 1, 700000), ([120000], 10, 50)])                   # clusters of 16, remade, and of 8
@pytest.mark.parametrize("ties", [False, True])
def test_evict_rounds(s3b, engine, lengths, heads, keep, ties):
    """Tokens whose threshold is found digit by digit, by one block or a cluster, with keys in shared memory and remade from the
    weights where more than 49152 tokens fall to a block."""
    s = Sequences(s3b, engine, 2, 64, heads, 16, lengths, seed=lengths[0], spare=len(lengths) * (keep // 16 + 1))
    check_evict(s3b, engine, s, some_weights(s, ties), keep, 4, 100 if keep > 104 else 0)


# ---------------------------------------------------------------- the longest lists
@pytest.mark.parametrize("call,keep", [("evict", 2 ** 31 - 1), ("evict", 2 ** 31 - 8191), ("select", 2 ** 31 - 1), ("select", 2 ** 27), ("select", 2 ** 27 - 511),
                                       ("attend", 2 ** 31 - 1), ("attend", 2 ** 27 - 511)])
def test_longer_lists_than_tokens_are_refused(raw, engine, call, keep):  # noqa: F811
    before = {name: x.clone() for name, x in raw.o.items() if x is not None}
    assert getattr(raw, call)(keep=keep) == -6
    engine.sync()
    for name, x in before.items():
        assert torch.equal(raw.o[name].view(torch.uint8), x.view(torch.uint8)), name


def test_the_longest_eviction(s3b, engine):
    """Room for 2^31 - 8192 kept positions of a short sequence: all behind the last are -1, and nothing around them is written."""
    needs(14)
    keep, guard, n, page = 2 ** 31 - 8192, 1 << 16, 40, 1 << 20
    s = Sequences(s3b, engine, 2, 64, 1, 16, [n], seed=1)
    to = s3b.KVCache(2, 1, page, 1, 64)
    around = torch.full((keep + 2 * guard,), 9, dtype=torch.int32, device="cuda")
    kept = around[guard:guard + keep].view(1, 1, keep)
    pages_out = torch.zeros(1, 2048, dtype=torch.int32, device="cuda")
    lengths_out = torch.zeros(1, dtype=torch.int32, device="cuda")
    engine.cache_evict(s.cache, torch.rand(1, 1, 48, device="cuda"), s.pages, s.lengths, pages_out, lengths_out, kept, to=to)
    engine.sync()
    assert lengths_out.item() == n and kept[0, 0, :n].tolist() == list(range(n))
    assert (around[:guard] == 9).all() and (around[guard + keep:] == 9).all()
    for i in range(n, keep, 2 ** 29):
        assert (kept[0, 0, i:i + 2 ** 29] == -1).all()
    k, v = s.rows(0)
    moved = [torch.empty_like(k) for _ in "kv"]
    engine.cache_read(to, torch.arange(n, device="cuda"), *moved)
    engine.sync()
    assert torch.equal(moved[0], k) and torch.equal(moved[1], v)


# ---------------------------------------------------------------- lengths that change meanwhile
@pytest.mark.parametrize("nq,d", [(1, 64), (9, 128), (9, 256), (30, 64), (30, 128), (200, 64), (200, 256)])
def test_weights_end_whatever_the_lengths_become(s3b, engine, nq, d):
    """Another stream writes the lengths while weights are gathered: what comes of it is the caller's, but the calls end, write nothing
    outside their rows, and leave later calls as they were."""
    lens = [(37 * i) % 900 for i in range(400)]
    e = s3b.Engine(0)  # on a stream of its own
    s = Sequences(s3b, engine, 2, d, 2, 16, lens, seed=nq)
    tokens = s.pages.shape[1] * 16
    around = torch.full((402, 2, tokens), 5.0, device="cuda")
    weights = around[1:401]
    q, lse = s.queries(nq, 4), torch.full((400, nq, 4), 4.0, device="cuda")
    others = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0] * 400, lens[::-1], [900] * 400, [16] * 399 + [0])]
    good, side = s.lengths.clone(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for i in range(60):
        e.cache_weights(s.cache, q, lse, weights, s.pages, s.lengths, 0.1, causal=bool(i % 2), window=50 if i % 4 == 3 else 0)
        with torch.cuda.stream(side):
            for x in others:
                s.lengths.copy_(x)
    torch.cuda.synchronize()
    e.close()
    assert (around[0] == 5).all() and (around[401] == 5).all()
    s.lengths.copy_(good)
    e = s3b.Engine(0)
    a, b = torch.zeros(400, 2, tokens, device="cuda"), torch.zeros(400, 2, tokens, device="cuda")
    torch.cuda.synchronize()
    e.cache_weights(s.cache, q, lse, a, s.pages, s.lengths, 0.1)
    for i in range(0, 400, 50):
        e.cache_weights(s.cache, q[i:i + 50], lse[i:i + 50], b[i:i + 50], s.pages[i:i + 50], s.lengths[i:i + 50], 0.1)
    e.sync()
    e.close()
    # where many CTAs share a tile its parts are cut elsewhere: f32 sums of at most 400 terms in another order
    assert (a - b).abs().max() <= 400 * 2.0 ** -24 * a.max()


# ---------------------------------------------------------------- arrays over each other
@pytest.mark.parametrize("off,refused", [(-3, False), (-2, True), (-1, True), (0, True), (1, True), (2, True), (3, False)])
def test_new_lengths_over_the_lengths_are_refused(s3b, engine, off, refused):
    """One sequence's new length would be read as another's."""
    s = Sequences(s3b, engine, 2, 64, 2, 16, [40, 33, 50], seed=2, spare=3)
    both = torch.full((9,), -5, dtype=torch.int32, device="cuda")
    both[3:6] = s.lengths
    kept = torch.full((3, 2, 10), 9, dtype=torch.int32, device="cuda")
    free = sorted(set(range(s.cache.n_pages)) - set(s.pages.flatten().tolist()))
    pages_out = torch.tensor(free[:3], dtype=torch.int32, device="cuda")[:, None]
    args = (s.cache, some_weights(s), s.pages, both[3:6], pages_out, both[3 + off:6 + off], kept)
    if refused:
        with pytest.raises(s3b.S3BError, match="over the lengths"):
            engine.cache_evict(*args)
        engine.sync()
        assert (kept == 9).all() and both[3:6].tolist() == s.lens
    else:
        engine.cache_evict(*args)
        engine.sync()
        assert both[3 + off:6 + off].tolist() == [10, 10, 10] and both[3:6].tolist() == s.lens and (kept < 50).all()


# ---------------------------------------------------------------- f32 outputs
@pytest.mark.parametrize("qtype", [2, 3, 8])
@pytest.mark.parametrize("d,heads,kv,nq,share", [(64, 8, 2, 9, 1), (64, 4, 1, 16, 8), (128, 4, 2, 8, 4), (128, 8, 1, 6, 2), (256, 2, 1, 20, 4), (256, 4, 2, 12, 6)])
def test_f32_outputs_keep_the_weights(s3b, engine, qtype, d, heads, kv, nq, share):
    """Weights and their products with the block scales keep 2^-22 and more on the way to an f32 output. Few tokens and small queries,
    so that the bound is far below f16's half step, 2^-11: the score's error E and ex2's as in test_kv_long_gpu.py, the weight and the
    product with a remainder each (2^-21), six accumulations of one group of 16 tokens (16 products and the sum before, each cut at
    2^-24 of the largest) and 16 warps' sums. In q4_1 a value enters in two terms (test_kv_long_gpu.py)."""
    s = Sequences(s3b, engine, qtype, d, kv, 16, [2, 3, 5, 9, 16], seed=d + nq)
    q, scale, group = s.queries(nq, heads, 0.1), 0.9 * d ** -0.5, heads // kv
    out, lse = torch.full(q.shape, 9.0, device="cuda"), torch.full(q.shape[:3], 9.0, device="cuda")
    selected = torch.zeros(5, -(-nq // share), kv, 2, dtype=torch.int32, device="cuda")
    selected[..., 1] = -1
    engine.cache_attention_selected(s.cache, q, out, selected, s.pages, s.lengths, scale, share=share, lse=lse)
    engine.sync()
    for b in range(5):
        for h in range(kv):
            want, _, want_lse, _ = plain_attention(s, q, torch.arange(s.lens[b], device="cuda"), b, h, 0, nq, False, 0, scale)
            k, v = (x[:, h].double() for x in s.rows(b))
            x = q[b, :, h * group:(h + 1) * group].reshape(-1, d).double()
            e = ((d + 16) * 2.0 ** -24 * scale * (x.abs() @ k.abs().T)).amax(1, keepdim=True)
            p = (x @ k.T * scale).softmax(-1)
            blocks = v.view(-1, d // 32, 32)
            size = v.abs()
            if qtype == 3:
                size = size + (blocks.abs().amax(-1) + 2 * (blocks.amax(-1) - blocks.amin(-1))).repeat_interleave(32, -1)
            err = (2 * torch.expm1(e) + 2.0 ** -19 + 2.0 ** -21 + (6 * 17 + 16) * 2.0 ** -24) * (p @ size) + 1e-30
            assert err.max() < 2.0 ** -14 * size.max()
            got = out[b, :, h * group:(h + 1) * group].reshape(-1, d).double()
            assert ((got - want).abs() <= err).all(), (b, h, ((got - want).abs() / err).max())
            assert ((lse[b, :, h * group:(h + 1) * group].reshape(-1) - want_lse).abs() <= 2 * e[:, 0] + 2.0 ** -18).all()
