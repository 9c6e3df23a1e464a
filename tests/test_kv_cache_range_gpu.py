"""Attention over the quantised cache where magnitudes, counts and lengths go to their ends, against 64-bit arithmetic on the
values that the cache holds.

What is rounded to fewer than 32 bits, u = 2^-11 relative each at most: with few query rows the weight, its product with
the block scale and an f16 output; with many the keys, the values, the weight and an f16 output. Each rounding is off by
u / sqrt(3) at most in the mean square. So the error's norm over a whole output is below sqrt(3) u / sqrt(3) = u with few
rows, and where the keys' roundings move the scores by no more than u / sqrt(3) (scores of deviation 1) below 1.16 u with many,
which the bounds below take with a quarter added: NORM[few], NORM[many]. Where single scores are large, so that one key's
rounding moves a weight by more, many rows are compared with the keys as they round them."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -11
NORM = {True: 1.25 * U, False: 1.45 * U}


def most_few(d):
    """Rows of a key / value head up to which the call counts as one of few rows."""
    return 16 if d == 256 else 32


def attend(s3b, engine, qtype, q, k, v, lengths, page=64, scale=None, causal=False, window=0, out_dtype=torch.float32):
    """Attention of q f16 [batch, nq, heads, d] over the caches of k, v [batch, n, kv heads, d] in pages of a shuffled table:
    the output, lse, and the keys and values held (f32)."""
    batch, n, kv, d = k.shape
    per = -(-n // page)
    cache = s3b.KVCache(qtype, batch * per, page, kv, d)
    cache.data.fill_(0xFF)
    g = torch.Generator(device="cuda").manual_seed(n)
    pages = torch.randperm(batch * per, device="cuda", generator=g).to(torch.int32).view(batch, per)
    at = torch.arange(n, device="cuda")
    held = []
    for b in range(batch):
        m = lengths[b]
        slots = pages[b].long()[at[:m] // page] * page + at[:m] % page
        engine.cache_write(cache, k[b, :m], v[b, :m], slots)
        rows = [torch.empty(m, kv, d, device="cuda") for _ in "kv"]
        engine.cache_read(cache, slots, *rows)
        held.append(rows)
    out = torch.empty(q.shape, device="cuda", dtype=out_dtype)
    lse = torch.empty(q.shape[:3], device="cuda")
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    engine.cache_attention(cache, q, out, pages, lens, d ** -0.5 if scale is None else scale, causal=causal, window=window, lse=lse)
    engine.sync()
    return out, lse, held


def exact(q, held, scale, causal=False, window=0, keys16=False):
    """Attention of one sequence's q [nq, heads, d] over the values held (keys16: the keys rounded to f16) in 64 bits: output,
    lse."""
    k, v = held[0].half().double() if keys16 else held[0].double(), held[1].double()
    nq, heads, d = q.shape
    n, kv, _ = k.shape
    group = heads // kv
    hi = torch.arange(nq, device="cuda")[:, None] + (n - nq + 1) if causal else torch.full((nq, 1), n, device="cuda")
    at = torch.arange(n, device="cuda")
    hide = (at >= hi) | ((at < hi - window) if window else False)
    out, lse = (torch.zeros(nq, heads, m, device="cuda", dtype=torch.float64) for m in (d, 1))
    for h in range(heads):
        s = (q[:, h].double() @ k[:, h // group].T * scale).masked_fill(hide, -math.inf)
        lse[:, h, 0] = s.logsumexp(-1)
        p = s.softmax(-1).nan_to_num(0.0)
        out[:, h] = p @ v[:, h // group]
    return out, lse[..., 0]


def lse_off(d, score):
    """How far f32 scores of this size may be off: d / 16 product steps, each kept to 2^-22, the scale and the logarithm."""
    return (d / 16 + 2) * 2.0 ** -22 * score


def off(x, y):
    return ((x.double() - y).norm() / y.norm()).item()


@pytest.mark.parametrize("qtype", [2, 3, 8])
@pytest.mark.parametrize("d,nq,group", [(64, 1, 1), (128, 1, 4), (128, 5, 4), (64, 8, 4), (256, 1, 2), (256, 5, 3), (128, 70, 2)])
def test_large_queries(s3b, engine, qtype, d, nq, group):
    """Queries of 2047 to 60000 and of one sign: 32 of them sum past f16's largest. The scale brings the scores back to a
    deviation of about 1, where f32 sums over d products keep them to 2^-20."""
    g = torch.Generator(device="cuda").manual_seed(d + nq)
    n, kv = 700, 2
    k, v = (torch.randn(1, n, kv, d, device="cuda", generator=g) for _ in "kv")
    q = 4096 + 2000 * torch.rand(1, nq, kv * group, d, device="cuda", generator=g)
    q[:, :, ::2] *= -1
    q[:, :, -1] *= 9.8
    q = q.half()
    scale = 1.0 / (5000 * math.sqrt(d))
    q[:, :, 0] = torch.randn(nq, d, device="cuda", generator=g).half()  # a small row beside large ones
    out, lse, held = attend(s3b, engine, qtype, q, k, v, [n], page=48, scale=scale)
    ref, ref_lse = exact(q[0], held[0], scale)
    few = nq * group <= most_few(d)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    # the last head's scores deviate by about 10: with many rows the keys' roundings move them by as much more
    heads = slice(None) if few else slice(0, -1)
    assert off(out[0][:, heads], ref[:, heads]) < NORM[few]
    if few:
        assert (lse[0] - ref_lse).abs().max() < 1e-3


def sink_and_tail(n, kv, d, depth, gen):
    """Keys and values [1, n, kv, d] and a query direction: token 5 scores `depth` more than the others, whose scores deviate by
    0.25, with q = 8 in channel 0 and 0.5 randn in the others and a scale of 1 / 8."""
    k = 0.5 * torch.randn(1, n, kv, d, device="cuda", generator=gen) * (64 / d) ** 0.5
    k[..., 0] = 0
    k[:, 5, :, 0] = depth
    v = 0.5 + 0.5 * torch.randn(1, n, kv, d, device="cuda", generator=gen)
    v[:, 5] = -1 - torch.rand(kv, d, device="cuda", generator=gen)
    return k, v


@pytest.mark.parametrize("qtype", [2, 3, 8])
@pytest.mark.parametrize("d,nq,group", [(64, 1, 1), (128, 1, 4), (64, 9, 2), (128, 8, 4), (256, 1, 2), (256, 4, 4), (128, 60, 1), (256, 30, 1)])
@pytest.mark.parametrize("size", [1e4, 1.0, 1e-2, 1e-3, 1e-4, "blocks", "late"])
def test_long_tail_of_values_of_any_size(s3b, engine, qtype, d, nq, group, size):
    """One token 12 nats above 131075 others, which hold 44% of the weight between them. The values are large, near 1 or small; of
    another size in each block of 32 channels; or, late, a thousand times larger in the last fifth than before."""
    g = torch.Generator(device="cuda").manual_seed(d + nq)
    n, kv = 131075, 1
    k, v = sink_and_tail(n, kv, d, 12.0, g)
    if size == "blocks":
        v *= torch.tensor([1e3, 1e-3, 1.0, 1e-2, 30.0, 1e-4, 1e4, 0.1], device="cuda")[:d // 32].repeat_interleave(32)
    elif size == "late":
        v[:, 4 * n // 5:] *= 1e3
        v *= 1e-3
    else:
        v *= size
    q = 0.5 * torch.randn(1, nq, kv * group, d, device="cuda", generator=g)
    q[..., 0] = 8
    q = q.half()
    out, lse, held = attend(s3b, engine, qtype, q, k, v, [n], scale=0.125)
    few = nq * group <= most_few(d)
    ref, ref_lse = exact(q[0], held[0], 0.125, keys16=not few)
    for c in range(0, d, 32):
        assert off(out[0][..., c:c + 32], ref[..., c:c + 32]) < NORM[few], c
    assert (lse[0] - ref_lse).abs().max() < 1e-5


@pytest.mark.parametrize("qtype", [2, 3, 8])
@pytest.mark.parametrize("d,nq,group,page", [(64, 1, 1, 16), (128, 1, 4, 48), (128, 5, 4, 16), (256, 1, 2, 64), (256, 10, 1, 16), (64, 50, 1, 16)])
@pytest.mark.parametrize("size", [3e4, 100.0, 1e-2, 1e-3, 1e-4])
def test_values_of_any_size(s3b, engine, qtype, d, nq, group, page, size):
    """The same precision, relative to the values, whatever their size: a few hundred tokens of ordinary scores, f32 outputs."""
    g = torch.Generator(device="cuda").manual_seed(nq)
    n = 300
    k, v = (torch.randn(1, n, 2, d, device="cuda", generator=g) for _ in "kv")
    q = torch.randn(1, nq, 2 * group, d, device="cuda", generator=g).half()
    out, lse, held = attend(s3b, engine, qtype, q, k, v * (size / 5), [n], page=page)
    ref, ref_lse = exact(q[0], held[0], d ** -0.5)
    assert off(out[0], ref) < NORM[nq * group <= most_few(d)]


@pytest.mark.parametrize("qtype", [2, 3, 8])
@pytest.mark.parametrize("d,nq", [(64, 1), (128, 2), (256, 1), (64, 40)])
def test_sink_in_each_of_many_sequences(s3b, engine, qtype, d, nq):
    """160 sequences, so that a block has a whole one and a warp a long share of it: a token 12 nats above 20000 others, which hold
    11% of the weight."""
    g = torch.Generator(device="cuda").manual_seed(d)
    batch, n, kv = 160, 20001, 1
    k1, v1 = sink_and_tail(n, kv, d, 12.0, g)
    k1, v1 = k1.half(), (v1 * 0.05).half()
    q = 0.5 * torch.randn(batch, nq, kv, d, device="cuda", generator=g)
    q[..., 0] = 8
    q = q.half()
    lengths = [n - 7 * b for b in range(batch)]
    out, lse, held = attend(s3b, engine, qtype, q, k1.expand(batch, -1, -1, -1), v1.expand(batch, -1, -1, -1), lengths, scale=0.125)
    few = nq <= most_few(d)
    for b in range(0, batch, 53):
        ref, ref_lse = exact(q[b], held[b], 0.125, keys16=not few)
        assert off(out[b], ref) < NORM[few], b
        assert (lse[b] - ref_lse).abs().max() < 1e-5


@pytest.mark.parametrize("qtype", [2, 3, 8])
@pytest.mark.parametrize("d,nq", [(64, 1), (64, 40), (128, 1), (128, 140), (256, 2), (256, 30), (256, 900)])
def test_scores_of_ten_digits(s3b, engine, qtype, d, nq):
    """Queries and keys near f16's largest, of either sign: scores past 2^31, whose f32 step is far more than 1. The row takes
    the token with the largest; rows of small queries beside it are as ever."""
    g = torch.Generator(device="cuda").manual_seed(nq)
    n = 300
    k = (30000 + 100 * torch.randperm(n, device="cuda", generator=g))[None, :, None, None].expand(1, n, 1, d).float()
    v = torch.randn(1, n, 1, d, device="cuda", generator=g)
    q = 1e-5 * torch.rand(1, nq, 1, d, device="cuda", generator=g)
    q[:, ::3] = 6e4
    q[:, 1::3] = -6e4
    q = q.half()
    out, lse, held = attend(s3b, engine, qtype, q, k, v, [n], page=16)
    few = nq <= most_few(d)
    ref, ref_lse = exact(q[0], held[0], d ** -0.5, keys16=not few)
    assert off(out[0], ref) < NORM[few]
    assert ((lse[0] - ref_lse).abs() <= lse_off(d, ref_lse.abs()) + 1e-5).all()
