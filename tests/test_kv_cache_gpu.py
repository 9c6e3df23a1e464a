"""The quantised key / value cache: writing, reading back and attention against plain implementations.

Writing and reading are compared bit for bit with the host quantisers. Attention is compared with 64-bit arithmetic on
the values that the cache stands for. Its tolerance is a bound on what the kernels round to f16, each to a relative
u = 2^-11: the keys (a score is off by at most D = u * scale * sum |q k|, so a weight by exp(2 D) over numerator and
denominator), the weights and their products with the block scale, the values, and the output, plus f16's subnormal
step for the weights: (2 D + 5 u) * sum p |v| + u |out| + 2^-25 * n * max |v|."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -11


def _rows(gen, n, heads, d, dtype=torch.float32):
    k = torch.randn(n, heads, d, device="cuda", generator=gen) * torch.exp(0.4 * torch.randn(heads, d, device="cuda", generator=gen))
    v = torch.randn(n, heads, d, device="cuda", generator=gen) + 0.3
    return (k + 0.5).to(dtype), v.to(dtype)


def _held(s3b, qtype, rows):
    """What the host quantisers make of rows [..., d], as f32 CUDA values."""
    x = rows.float().cpu().numpy()
    y = s3b.dequantize_rows(qtype, s3b.quantize_rows(qtype, x.reshape(-1, x.shape[-1])), x.shape[-1])
    return torch.from_numpy(y.reshape(x.shape)).cuda()


def _read(engine, cache, slots, dtype=torch.float32):
    outs = [torch.full((len(slots), cache.heads, cache.d), 7.0, device="cuda", dtype=dtype) for _ in "kv"]
    engine.cache_read(cache, slots, *outs)
    engine.sync()
    return outs


# ---------------------------------------------------------------- write, read
@pytest.mark.parametrize("qtype", [2, 3, 8])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n,heads,page,src,dst", [(1, 1, 16, "f32", "f32"), (37, 3, 48, "f16", "f16"),
                                                  (37, 3, 48, "f32", "f16"), (515, 2, 64, "f16", "f32"), (16, 8, 16, "f32", "f32")])
def test_round_trip_matches_host(s3b, engine, qtype, d, n, heads, page, src, dst):
    g = torch.Generator(device="cuda").manual_seed(n * d + heads)
    pages = -(-n // page) + 2
    cache = s3b.KVCache(qtype, pages, page, heads, d)
    cache.data.fill_(0xA5)
    k, v = _rows(g, n, heads, d, torch.float16 if src == "f16" else torch.float32)
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:n].contiguous()
    engine.cache_write(cache, k, v, slots)
    dt = torch.float16 if dst == "f16" else torch.float32
    for got, rows in zip(_read(engine, cache, slots, dt), (k, v)):
        assert torch.equal(got, _held(s3b, qtype, rows).to(dt))


@pytest.mark.parametrize("qtype", [2, 3, 8])
def test_write_leaves_other_slots(s3b, engine, qtype):
    """Tokens written one by one, in any order, give the bytes of one call; skipped tokens and other slots keep theirs."""
    g = torch.Generator(device="cuda").manual_seed(qtype)
    d, heads, page = 128, 2, 32
    k, v = _rows(g, 40, heads, d)
    slots = torch.randperm(3 * page, device="cuda", generator=g)[:40].contiguous()
    a, b = (s3b.KVCache(qtype, 3, page, heads, d) for _ in "ab")
    for c in (a, b):
        c.data.fill_(0x5A)
    engine.cache_write(a, k, v, slots)
    for i in torch.randperm(40).tolist():
        engine.cache_write(b, k[i:i + 1], v[i:i + 1], slots[i:i + 1])
    engine.sync()
    assert torch.equal(a.data, b.data)
    engine.cache_write(b, k + 1, v + 1, torch.full_like(slots, -1))
    engine.sync()
    assert torch.equal(a.data, b.data)
    free = torch.tensor(sorted(set(range(3 * page)) - set(slots.tolist())), device="cuda")
    c = s3b.KVCache(qtype, 3, page, heads, d)
    c.data.fill_(0x5A)
    for x, y in zip(_read(engine, a, free), _read(engine, c, free)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("qtype", [2, 3, 8])
def test_write_odd_blocks(s3b, engine, qtype):
    """Blocks of equal values, of zeros, with equal magnitudes of both signs, with ties between two codes, tiny and huge."""
    d = 64
    x = torch.zeros(12, 1, d, device="cuda")
    x[1] = 3.25
    x[2] = -3.25
    x[3, 0, 5], x[3, 0, 9] = 4.0, -4.0
    x[4, 0, 5], x[4, 0, 9] = -4.0, 4.0
    x[5] = torch.arange(64, device="cuda") * 0.5 - 16
    x[6] = (torch.arange(64, device="cuda") * 0.5 - 16) * 1e-7
    x[7] = 1e-39
    x[8, 0, 0] = 65024.0
    x[9] = torch.linspace(-65024, 65024, 64, device="cuda")
    x[10] = torch.arange(64, device="cuda") % 2 * 2.0 - 1
    x[11] = torch.arange(64, device="cuda") * 127 / 63
    cache = s3b.KVCache(qtype, 1, 16, 1, d)
    slots = torch.arange(12, device="cuda")
    engine.cache_write(cache, x, -x, slots)
    for got, rows in zip(_read(engine, cache, slots), (x, -x)):
        assert torch.equal(got, _held(s3b, qtype, rows))
    for got in _read(engine, cache, slots, torch.float16):
        assert torch.isfinite(got).all()


@pytest.mark.parametrize("qtype", [2, 3, 8])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_write_holds_what_is_not_finite(s3b, engine, qtype, dtype):
    g = torch.Generator(device="cuda").manual_seed(9)
    k, v = _rows(g, 3, 1, 64, dtype)
    k[0, 0, 3], k[0, 0, 40], v[1, 0, 2], v[2, 0, 63] = math.inf, math.nan, -math.inf, math.nan
    if dtype == torch.float32:
        k[2, 0, 1] = 1e30
    cache = s3b.KVCache(qtype, 1, 16, 1, 64)
    slots = torch.arange(3, device="cuda")
    engine.cache_write(cache, k, v, slots)
    for got, rows in zip(_read(engine, cache, slots), (k, v)):
        assert torch.equal(got, _held(s3b, qtype, torch.nan_to_num(rows.float(), nan=0.0).clamp(-65024, 65024)))
    for got in _read(engine, cache, slots, torch.float16):
        assert torch.isfinite(got).all()


def test_strided_rows(s3b, engine):
    """k and v as slices of one fused projection, outputs as slices of a wider buffer, one output left out."""
    g = torch.Generator(device="cuda").manual_seed(3)
    n, heads, d = 21, 3, 64
    fused = torch.randn(n, 2 * heads * d + 8, device="cuda", generator=g).half()
    k = fused[:, :heads * d].view(n, heads, d)
    v = fused[:, heads * d:2 * heads * d].unflatten(1, (d // 8, heads, 8)).transpose(1, 2).reshape(n, heads, d)
    v = torch.empty(heads, n, d, device="cuda", dtype=torch.float16).copy_(v.transpose(0, 1)).transpose(0, 1)
    cache = s3b.KVCache(2, 2, 16, heads, d)
    slots = torch.arange(3, 3 + n, device="cuda")
    engine.cache_write(cache, k, v, slots)
    wide = torch.full((n, heads, 2 * d), 9.0, device="cuda")
    engine.cache_read(cache, slots, wide[:, :, d:], None)
    engine.sync()
    assert torch.equal(wide[:, :, d:], _held(s3b, 2, k)) and (wide[:, :, :d] == 9).all()
    engine.cache_read(cache, slots, None, wide[:, :, :d])
    engine.sync()
    assert torch.equal(wide[:, :, :d], _held(s3b, 2, v)) and torch.equal(wide[:, :, d:], _held(s3b, 2, k))


def test_skipped_and_empty_reads(s3b, engine):
    g = torch.Generator(device="cuda").manual_seed(4)
    cache = s3b.KVCache(3, 1, 16, 2, 128)
    k, v = _rows(g, 16, 2, 128)
    engine.cache_write(cache, k, v, torch.arange(16, device="cuda"))
    kk, vv = _read(engine, cache, torch.tensor([5, -1, 0, -7], device="cuda"))
    assert torch.equal(kk[[0, 2]], _held(s3b, 3, k[[5, 0]])) and torch.equal(vv[[0, 2]], _held(s3b, 3, v[[5, 0]]))
    assert not kk[[1, 3]].any() and not vv[[1, 3]].any()
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    engine.cache_write(cache, k[:0], v[:0], none)
    assert _read(engine, cache, none)[0].shape[0] == 0


# ---------------------------------------------------------------- attention
def _spans(n, nq, causal, window):
    hi = [n - nq + i + 1 if causal else n for i in range(nq)]
    return [(max(0, h - window) if window else 0, max(h, 0)) for h in hi]


def _check(s3b, engine, qtype, d, heads, kv, nq, lengths, page, causal=False, window=0, out_dtype=torch.float16, fill=0xFF,
           spare=3, q_scale=1.0, check=None):
    """Attention over sequences written into shuffled pages of a cache whose other bytes are `fill` (0xFF: NaN scales)."""
    g = torch.Generator(device="cuda").manual_seed(d * 7 + heads * 3 + nq + sum(lengths))
    batch, per = len(lengths), max(1, -(-max(lengths) // page))
    total = batch * per + spare
    cache = s3b.KVCache(qtype, total, page, kv, d)
    cache.data.fill_(fill)
    order = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    pages = torch.full((batch, per + 1), -1, dtype=torch.int32, device="cuda")  # entries past a sequence's pages are not read
    held = []
    for b, n in enumerate(lengths):
        used = -(-n // page)
        pages[b, :used] = order[b * per:b * per + used]
        at = torch.arange(n, device="cuda")
        slots = pages[b].long()[at // page] * page + at % page
        k, v = _rows(g, n, kv, d)
        engine.cache_write(cache, k, v, slots)
        held.append((_held(s3b, qtype, k).double(), _held(s3b, qtype, v).double()) if n else None)
    q = (torch.randn(batch, nq, heads, d, device="cuda", generator=g) * q_scale).half()
    out = torch.full((batch, nq, heads, d), 5.0, device="cuda", dtype=out_dtype)
    lse = torch.full((batch, nq, heads), 5.0, device="cuda")
    scale = d ** -0.5
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    engine.cache_attention(cache, q, out, pages[:, :per], lens, scale, causal=causal, window=window, lse=lse)
    engine.sync()
    again, lse2 = torch.empty_like(out), torch.empty_like(lse)
    engine.cache_attention(cache, q, again, pages[:, :per], lens, scale, causal=causal, window=window, lse=lse2)
    engine.sync()
    assert torch.equal(out, again) and torch.equal(lse, lse2)  # no result depends on the order of blocks
    group = heads // kv
    for b, n in enumerate(lengths):
        spans = _spans(n, nq, causal, window)
        empty = torch.tensor([hi <= lo for lo, hi in spans], device="cuda")
        assert not out[b][empty].any() and (lse[b][empty] == -math.inf).all()
        if empty.all():
            continue
        k, v = (t.repeat_interleave(group, 1) for t in held[b])
        at = torch.arange(n, device="cuda")
        lo, hi = (torch.tensor(x, device="cuda")[:, None, None] for x in zip(*spans))
        see = (at >= lo) & (at < hi)                                             # [nq, 1, n]
        qb = q[b].double()
        s = torch.einsum("ihd,nhd->ihn", qb, k) * scale
        off = (torch.einsum("ihd,nhd->ihn", qb.abs(), k.abs()) * scale * U).masked_fill(~see, 0).amax(-1)[..., None]
        p = s.masked_fill(~see, -math.inf).softmax(-1).nan_to_num(0.0)
        ref = torch.einsum("ihn,nhd->ihd", p, v)
        tol = (2 * off + 5 * U) * torch.einsum("ihn,nhd->ihd", p, v.abs()) + U * ref.abs() + 2.0 ** -25 * n * v.abs().max()
        bad = ((out[b].double() - ref).abs() > tol) & ~empty[:, None, None]
        assert not bad.any(), (b, n, (out[b].double() - ref).abs().max().item(), tol.max().item(), bad.nonzero()[:4].tolist())
        ref_lse = s.masked_fill(~see, -math.inf).logsumexp(-1)
        err = (lse[b].double() - ref_lse).abs()[~empty]
        assert (err <= off[..., 0][~empty] + 4 * U).all(), err.max().item()


CASES = [  # d, heads, kv heads, nq, lengths, page, causal, window
    (64, 1, 1, 1, [1], 16, False, 0),
    (64, 8, 8, 1, [577], 16, False, 0),
    (128, 4, 1, 1, [0, 1, 15, 16, 17, 31, 300, 0], 16, False, 0),
    (128, 24, 3, 1, [130, 2049, 64], 48, False, 0),
    (256, 1, 1, 1, [1111, 90], 64, False, 0),
    (256, 6, 2, 3, [700, 2, 0, 3], 80, True, 0),
    (64, 12, 4, 5, [200, 3, 64, 0, 5], 48, True, 70),
    (128, 8, 8, 7, [333, 6, 1], 32, True, 16),
    (128, 2, 1, 1, [5000], 64, True, 128),
    (64, 16, 1, 1, [900, 1], 16, False, 0),
    (128, 16, 2, 2, [600, 77], 16, False, 0),
    (64, 2, 2, 130, [300, 129, 0, 40], 32, True, 0),
    (128, 4, 2, 200, [450, 200], 16, True, 0),
    (128, 3, 1, 65, [1000, 1], 64, False, 0),
    (256, 2, 1, 150, [777, 60], 48, True, 100),
    (256, 1, 1, 300, [900], 64, False, 0),
    (64, 5, 5, 257, [515], 16, True, 33),
]


@pytest.mark.parametrize("qtype", [2, 3, 8])
@pytest.mark.parametrize("d,heads,kv,nq,lengths,page,causal,window", CASES)
def test_attention(s3b, engine, qtype, d, heads, kv, nq, lengths, page, causal, window):
    _check(s3b, engine, qtype, d, heads, kv, nq, lengths, page, causal, window)


@pytest.mark.parametrize("nq", [1, 4, 9, 17, 33, 64, 100, 128, 129])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_query_counts(s3b, engine, d, nq):
    _check(s3b, engine, 2, d, 3, 1, nq, [260, nq + 1, 19], 32, True, out_dtype=torch.float32)


@pytest.mark.parametrize("qtype,d,page", [(2, 256, 16), (8, 256, 64), (3, 128, 48), (2, 64, 16)])
def test_attention_many_row_blocks(s3b, engine, qtype, d, page):
    """Uneven sequences of several row blocks each: every share of the work begins and ends inside one."""
    _check(s3b, engine, qtype, d, 4, 2, 600, [1200, 901, 33, 1100, 640, 1025], page, True)


@pytest.mark.parametrize("nq", [1, 140])
@pytest.mark.parametrize("qtype", [2, 8])
def test_attention_peaked(s3b, engine, qtype, nq):
    """Large queries: the weight sits on single tokens, and the running maximum moves late in the sequence."""
    _check(s3b, engine, qtype, 128, 4, 2, nq, [700, 160], 16, causal=nq > 1, q_scale=30.0)


@pytest.mark.parametrize("nq", [1, 64, 256])
def test_attention_of_masked_extremes(s3b, engine, nq):
    """Tokens that a mask hides hold the largest values that a cache takes: no other row may feel them."""
    d, page, n = 128, 16, 400
    g = torch.Generator(device="cuda").manual_seed(nq)
    cache = s3b.KVCache(2, 40, page, 1, d)
    k, v = _rows(g, n, 1, d)
    pages = torch.arange(25, dtype=torch.int32, device="cuda")[None]
    slots = torch.arange(n, device="cuda")
    q = torch.randn(1, nq, 2, d, device="cuda", generator=g).half()
    outs = []
    for wild in (False, True):
        if wild:  # the last token is seen by the last query only
            k[-1], v[-1] = math.inf, -math.inf
        engine.cache_write(cache, k, v, slots)
        out = torch.empty_like(q)
        engine.cache_attention(cache, q, out, pages, torch.tensor([n], dtype=torch.int32, device="cuda"), d ** -0.5, causal=True)
        engine.sync()
        outs.append(out)
    assert torch.equal(outs[0][:, :-1], outs[1][:, :-1]) and torch.isfinite(outs[1]).all()


def test_attention_strides_and_stream(s3b, engine):
    """q inside a fused projection, out inside a wider buffer, a page table with spare columns, on a stream of its own."""
    g = torch.Generator(device="cuda").manual_seed(5)
    d, heads, kv, nq, n, page = 64, 4, 2, 3, 100, 16
    cache = s3b.KVCache(3, 8, page, kv, d)
    k, v = _rows(g, n, kv, d)
    table = torch.arange(16, dtype=torch.int32, device="cuda").view(2, 8)
    table[1] = table[0]
    fused = torch.randn(2, nq, heads * d + 64, device="cuda", generator=g).half()
    q = fused[..., :heads * d].unflatten(-1, (heads, d))
    wide = torch.full((2, heads, nq, 2 * d), 3.0, device="cuda")
    out = wide.transpose(1, 2)[..., d:]
    lens = torch.tensor([n, 50], dtype=torch.int32, device="cuda")
    plain = torch.empty(2, nq, heads, d, device="cuda")
    engine.cache_write(cache, k, v, torch.arange(n, device="cuda"))
    engine.cache_attention(cache, q.contiguous(), plain, table[:, :7].contiguous(), lens, 0.125, causal=True)
    engine.sync()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    other = s3b.Engine(0)
    other.set_stream(stream.cuda_stream)
    other.cache_attention(cache, q, out, table[:, :7], lens, 0.125, causal=True)
    other.sync()
    other.close()
    assert torch.equal(out, plain) and (wide[..., :d] == 3).all()


def test_cache_past_32_bits(s3b, engine):
    """Slots whose bytes lie past 2^32."""
    d, heads, page = 256, 16, 64
    pages = (5 << 30) // s3b.kv_cache_bytes(8, heads, d, page, 1)
    cache = s3b.KVCache(8, pages, page, heads, d, data=torch.empty(s3b.kv_cache_bytes(8, heads, d, page, pages), dtype=torch.uint8, device="cuda"))
    g = torch.Generator(device="cuda").manual_seed(6)
    n = 3 * page
    k, v = _rows(g, n, heads, d)
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device="cuda")
    at = torch.arange(n, device="cuda")
    slots = table[0].long()[at // page] * page + at % page
    engine.cache_write(cache, k, v, slots)
    for got, rows in zip(_read(engine, cache, slots), (k, v)):
        assert torch.equal(got, _held(s3b, 8, rows))
    small = s3b.KVCache(8, 3, page, heads, d)
    engine.cache_write(small, k, v, at)
    lens = torch.tensor([n - 5], dtype=torch.int32, device="cuda")
    for nq in (1, 130):
        q = torch.randn(1, nq, heads, d, device="cuda", generator=g).half()
        a, b = torch.empty_like(q), torch.empty_like(q)
        engine.cache_attention(cache, q, a, table, lens, 0.0625)
        engine.cache_attention(small, q, b, torch.arange(3, dtype=torch.int32, device="cuda")[None], lens, 0.0625)
        engine.sync()
        assert torch.equal(a, b)


# ---------------------------------------------------------------- refusals
def test_refusals(s3b, engine):
    cache = s3b.KVCache(2, 4, 16, 2, 64)
    k = torch.zeros(3, 2, 64, device="cuda")
    slots = torch.arange(3, device="cuda")
    q = torch.zeros(1, 1, 4, 64, device="cuda", dtype=torch.float16)
    out = torch.empty_like(q)
    pages = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    lens = torch.tensor([3], dtype=torch.int32, device="cuda")

    def refuses(call, *args, **kw):
        with pytest.raises(s3b.S3BError):
            call(*args, **kw)

    refuses(engine.cache_write, cache, k, k.half(), slots)
    refuses(engine.cache_write, cache, k.double(), k.double(), slots)
    refuses(engine.cache_write, cache, k[:2], k, slots)
    refuses(engine.cache_write, cache, k, k, slots.int())
    refuses(engine.cache_write, cache, torch.zeros(3, 2, 65, device="cuda")[..., 1:], k, slots)  # rows off 16 bytes
    refuses(engine.cache_write, cache, torch.zeros(3, 2, 128, device="cuda")[..., ::2], k, slots)
    refuses(engine.cache_read, cache, slots, k, k.half())
    refuses(engine.cache_attention, cache, q.float(), out, pages, lens, 0.1)
    refuses(engine.cache_attention, cache, q[..., :3, :], out[..., :3, :], pages, lens, 0.1)  # 3 heads over 2
    refuses(engine.cache_attention, cache, q, out[:, :, :2], pages, lens, 0.1)
    refuses(engine.cache_attention, cache, q, out, pages.long(), lens, 0.1)
    refuses(engine.cache_attention, cache, q, out, pages, lens.long(), 0.1)
    # tensors that are not on the GPU
    refuses(s3b.KVCache, 2, 4, 16, 2, 64, device="cpu")
    refuses(engine.cache_write, cache, k.cpu(), k, slots)
    refuses(engine.cache_write, cache, k, k, slots.cpu())
    refuses(engine.cache_read, cache, slots, None, k.cpu())
    refuses(engine.cache_attention, cache, q.cpu(), out, pages, lens, 0.1)
    refuses(engine.cache_attention, cache, q, out.cpu(), pages, lens, 0.1)
    refuses(engine.cache_attention, cache, q, out, pages.cpu(), lens, 0.1)
    refuses(engine.cache_attention, cache, q, out, pages, lens.cpu(), 0.1)
    refuses(engine.cache_attention, cache, q, out, pages, lens, 0.1, lse=torch.empty(1, 1, 4))
    for scale in (0.0, -1.0, math.inf, math.nan):
        refuses(engine.cache_attention, cache, q, out, pages, lens, scale)
    refuses(engine.cache_attention, cache, q, out, pages, lens, 0.1, window=4)
    refuses(engine.cache_attention, cache, q, out, pages, lens, 0.1, causal=True, window=-4)
    refuses(s3b.KVCache, 2, 4, 16, 2, 64, data=torch.zeros(16, dtype=torch.uint8, device="cuda"))
    bad = s3b.KVCache(2, 4, 16, 2, 64)
    for field, value in (("type", 1), ("d", 96), ("heads", 0), ("page_size", 20), ("n_pages", 0), ("data", None),
                         ("data", cache.data.data_ptr() + 8)):
        bad.desc = s3b.KVCacheDesc(2, 2, 64, 16, 4, cache.data.data_ptr())
        setattr(bad.desc, field, value)
        rc = engine._L.s3b_op_cache_write(engine.h, bad.desc, k.data_ptr(), 128, 64, k.data_ptr(), 128, 64, 0, slots.data_ptr(), 3)
        assert rc == -1, field
    L, d = engine._L, cache.desc
    assert L.s3b_op_cache_write(engine.h, None, k.data_ptr(), 128, 64, k.data_ptr(), 128, 64, 0, slots.data_ptr(), 3) == -1
    assert L.s3b_op_cache_write(engine.h, d, None, 128, 64, k.data_ptr(), 128, 64, 0, slots.data_ptr(), 3) == -1
    assert L.s3b_op_cache_write(engine.h, d, k.data_ptr(), 128, 64, k.data_ptr(), 128, 64, 2, slots.data_ptr(), 3) == -6
    assert L.s3b_op_cache_write(engine.h, d, k.data_ptr(), 128, 64, k.data_ptr(), 128, 64, 0, slots.data_ptr(), -1) == -1
    assert L.s3b_op_cache_read(engine.h, d, None, 3, k.data_ptr(), 128, 64, None, 0, 0, 0) == -1
    engine.sync()


def test_index_errors_are_reported(s3b, engine):
    """Indexes in device memory that lie outside the cache are skipped or clamped, and the next sync says so."""
    g = torch.Generator(device="cuda").manual_seed(8)
    cache = s3b.KVCache(2, 4, 16, 1, 64)
    before = cache.data.clone()
    k, v = _rows(g, 2, 1, 64)

    def reports():
        with pytest.raises(s3b.S3BError, match="out of range"):
            engine.sync()
        engine.sync()  # reported once, the context goes on

    engine.cache_write(cache, k, v, torch.tensor([64, 1 << 40], device="cuda"))
    reports()
    assert torch.equal(cache.data, before)
    outs = [torch.full((1, 1, 64), 4.0, device="cuda") for _ in "kv"]
    engine.cache_read(cache, torch.tensor([64], device="cuda"), *outs)
    reports()
    assert not outs[0].any() and not outs[1].any()
    for nq in (1, 140):
        q = torch.zeros(1, nq, 1, 64, device="cuda", dtype=torch.float16)
        out = torch.empty_like(q)
        for page, n in ((4, 16), (-1, 16), (1, 17), (1, -1)):
            engine.cache_attention(cache, q, out, torch.tensor([[page]], dtype=torch.int32, device="cuda"),
                                   torch.tensor([n], dtype=torch.int32, device="cuda"), 0.1)
            reports()
