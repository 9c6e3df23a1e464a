"""Attention over the quantised cache in every block shape of its kernels: many units and sequences, long sequences in many
parts, staged and unstaged operands; each token counted exactly once."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_kv_cache_range_gpu import NORM, U, exact, lse_off, most_few  # noqa: E402


def _paged(s3b, engine, qtype, k, v, page, gen, spare=2):
    """A cache with the tokens k, v [n, kv, d] in shuffled pages, its other bytes NaN scales: cache, page row, values held."""
    n, kv, d = k.shape
    per = -(-n // page)
    cache = s3b.KVCache(qtype, per + spare, page, kv, d)
    cache.data.fill_(0xFF)
    row = torch.randperm(per + spare, device="cuda", generator=gen)[:per].to(torch.int32)
    at = torch.arange(n, device="cuda")
    slots = row.long()[at // page] * page + at % page
    engine.cache_write(cache, k, v, slots)
    held = [torch.empty(n, kv, d, device="cuda") for _ in "kv"]
    engine.cache_read(cache, slots, *held)
    return cache, row, held


def _compare(q, out, lse, held, lengths, causal, window, few, qtype):
    """Sequence by sequence: an element is off by u sum p (|v| + |w|) at most (5% more for f32 steps), from the rounding of the
    weight and from that of its product with the scale or of the value, and all of them by their norm. w is what the second
    rounding is relative to: v, but with few rows in q4_1 scale * (code - 8), the values less their block's middle."""
    d = q.shape[-1]
    errs, refs = [], []
    rounded = held[1]
    if few and qtype == 3:
        block = held[1].unflatten(-1, (-1, 32))
        low, high = block.amin(-1, keepdim=True), block.amax(-1, keepdim=True)  # codes 0 and 15
        rounded = (block - (low + 8 * (high - low) / 15)).flatten(-2)
    for b in range(len(lengths)):
        n = lengths[b]
        if n == 0:
            assert not out[b].any() and (lse[b] == -math.inf).all()
            continue
        own = [t[:n] for t in held]
        ref, ref_lse = exact(q[b], own, d ** -0.5, causal, window, keys16=not few)
        size, _ = exact(q[b], (own[0], own[1].abs() + rounded[:n].abs()), d ** -0.5, causal, window, keys16=not few)
        err = out[b].double() - ref
        bad = err.abs() > 1.05 * U * size
        assert not bad.any(), (b, n, bad.nonzero()[:4].tolist(), err.abs().max().item())
        seen = ref_lse > -math.inf
        assert torch.equal(lse[b] > -math.inf, seen)
        assert ((lse[b].double() - ref_lse)[seen].abs() <= lse_off(d, 10.0)).all(), (b, n)
        errs.append(err.flatten())
        refs.append(ref.flatten())
    assert (torch.cat(errs).norm() / torch.cat(refs).norm()).item() < NORM[few]


@pytest.mark.parametrize("qtype", [2, 3, 8])
@pytest.mark.parametrize("d,kv,group,nq,batch,page,causal,window", [
    # units for four-warp blocks (from 148 on), 8, 16 and 32 rows; sequences past the first 32
    (64, 3, 4, 1, 67, 16, False, 0), (64, 2, 4, 3, 100, 48, True, 90), (64, 5, 8, 4, 33, 32, True, 0),
    (128, 8, 4, 1, 41, 64, False, 0), (128, 2, 4, 4, 90, 16, True, 0), (128, 2, 8, 4, 75, 16, True, 200),
    (256, 1, 8, 1, 160, 16, False, 0), (256, 2, 4, 4, 77, 48, True, 0),
    # blocks of an SM each over many short sequences
    (64, 1, 2, 1, 140, 16, False, 0), (128, 1, 16, 1, 60, 32, False, 0), (256, 1, 5, 3, 100, 16, True, 40),
    # many rows: more pairs of sequence and row block than warps, some without a token
    (64, 2, 2, 40, 70, 16, True, 0), (128, 1, 4, 70, 100, 16, True, 64), (256, 1, 1, 150, 60, 32, True, 0),
])
def test_many_sequences(s3b, engine, qtype, d, kv, group, nq, batch, page, causal, window):
    g = torch.Generator(device="cuda").manual_seed(d + batch)
    most = 700
    k, v = (torch.randn(most, kv, d, device="cuda", generator=g) for _ in "kv")
    cache, row, held = _paged(s3b, engine, qtype, k, v, page, g)
    lengths = [(b * 7919 + 13) % (most + 1) if b % 9 else (0, 1, 16, most)[b // 9 % 4] for b in range(batch)]
    q = torch.randn(batch, nq, kv * group, d, device="cuda", generator=g).half()
    out, lse = torch.full(q.shape, 9.0, device="cuda"), torch.full(q.shape[:3], 9.0, device="cuda")
    engine.cache_attention(cache, q, out, row.expand(batch, -1).contiguous(), torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                           d ** -0.5, causal=causal, window=window, lse=lse)
    engine.sync()
    _compare(q, out, lse, held, lengths, causal, window, nq * group <= most_few(d), qtype)


@pytest.mark.parametrize("qtype", [2, 3, 8])
@pytest.mark.parametrize("d,kv,group,nq,n,causal,window", [
    (64, 1, 1, 1, 130001, False, 0), (128, 2, 8, 1, 100003, False, 0), (256, 1, 4, 1, 110017, False, 0), (128, 1, 4, 8, 120000, True, 70001),
    (64, 1, 4, 20, 100100, True, 0), (128, 1, 2, 64, 100100, True, 0), (256, 1, 1, 200, 100100, False, 0),
    # staged operands
    (64, 1, 2, 400, 20011, True, 0), (128, 2, 2, 500, 10007, True, 0), (128, 1, 1, 900, 9001, True, 3001), (256, 1, 1, 900, 12345, True, 0),
    (256, 1, 2, 700, 9000, False, 0),
])
def test_long_sequences(s3b, engine, qtype, d, kv, group, nq, n, causal, window):
    g = torch.Generator(device="cuda").manual_seed(d + n)
    k, v = (torch.randn(n, kv, d, device="cuda", generator=g) for _ in "kv")
    cache, row, held = _paged(s3b, engine, qtype, k, v, 64, g)
    q = torch.randn(1, nq, kv * group, d, device="cuda", generator=g).half()
    out, lse = torch.full(q.shape, 9.0, device="cuda"), torch.full(q.shape[:3], 9.0, device="cuda")
    engine.cache_attention(cache, q, out, row[None], torch.tensor([n], dtype=torch.int32, device="cuda"), d ** -0.5, causal=causal,
                           window=window, lse=lse)
    engine.sync()
    _compare(q, out, lse, held, [n], causal, window, nq * group <= most_few(d), qtype)


@pytest.mark.parametrize("qtype,page", [(2, 16), (3, 48), (8, 64)])
@pytest.mark.parametrize("d,kv,rows", [(64, 1, 1), (64, 3, 20), (128, 2, 8), (128, 1, 30), (256, 1, 16), (64, 1, 60), (128, 2, 200), (256, 1, 90),
                                       (64, 1, 700), (128, 1, 800), (256, 1, 900)])
@pytest.mark.parametrize("n", [1, 16, 33, 127, 129, 511, 513, 1025, 4097, 20001, 150001])
def test_every_token_counts_once(s3b, engine, qtype, page, d, kv, rows, n):
    """Queries of zero weigh all tokens alike: lse is ln n (f32 keeps a token more or less in 150001 apart), and a channel in which
    one token alone has a value gives that value / n. The tokens are at the ends of groups, tiles, pages and shares."""
    g = torch.Generator(device="cuda").manual_seed(n + d)
    tokens = torch.cat([torch.tensor([0, n - 1], device="cuda"), torch.randint(0, max(1, n // page), (d // 4,), device="cuda", generator=g) * page,
                        torch.randint(0, max(1, n // 128), (d // 4,), device="cuda", generator=g) * 128 - 1,
                        torch.randint(0, n, (d,), device="cuda", generator=g)])[:d].clamp(0, n - 1)
    k, v = torch.randn(n, kv, d, device="cuda", generator=g), torch.zeros(n, kv, d, device="cuda")
    v[tokens, :, torch.arange(d, device="cuda")] = 1.0
    cache, row, held = _paged(s3b, engine, qtype, k, v, page, g)
    q = torch.zeros(1, rows, kv, d, device="cuda", dtype=torch.float16)
    out, lse = torch.full(q.shape, 9.0, device="cuda"), torch.full(q.shape[:3], 9.0, device="cuda")
    engine.cache_attention(cache, q, out, row[None], torch.tensor([n], dtype=torch.int32, device="cuda"), 1.0, lse=lse)
    engine.sync()
    assert (lse.double() - math.log(n)).abs().max() < 4e-6
    want = held[1].double().sum(0) / n
    assert ((out[0].double() - want).abs() <= 2.1 * U * want.abs()).all()
