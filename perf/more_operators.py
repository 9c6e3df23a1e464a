"""Cases of the operators for caches longer than a step should read: bounds of each page's keys, a choice of pages by a
cheap score, attention over the chosen pages, the attention weight that each token has gathered, and eviction by it.

The cache is the quantised one (q4_0, q4_1 or q8_0 blocks of 32 values with float16 scales and minima), in pages of 16 or
more tokens that a sequence takes from its row of a page table. Query head h reads key/value head h // (heads / kv_heads).
With `causal` query i of nq is the token at position length - nq + i and sees no later one; with `window` > 0 only the last
`window` positions up to its own.

  bounds   per page, head and channel the least and the largest key (as float16, over the page's tokens), in 8 bits rounded
           outward: step = max |key| / 127, low = floor(key / step), high = ceil(key / step)
  select   blocks of `share` queries take `keep` pages each. A row's query in 8 bits c = round(q / t), t = max |q| / 127; its
           score of a page (sum over channels of max(c * low, c * high)) * step * t, a bound of q k up to the rounding of q;
           a block's score the largest of its rows (share x the heads of a group). The first `sink` and the last `recent`
           pages that the block sees are taken, then those of highest score, the lower page first among equals.
  attend   out = softmax(scale q k^T) v over the tokens of the chosen pages, and ln sum exp
  weights  w[token] = decay * w[token] + sum over rows of exp(scale q k - lse)
  evict    of each head the first `sink` and last `recent` tokens and those of highest weight, the earlier first among
           equals, `keep` in all, are moved in order to other pages
"""
import math

import torch

own = False

QTYPES = {"q4_0": 2, "q4_1": 3, "q8_0": 8}
LIMIT = 65024.0  # magnitude that a value is held to before it is quantised


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a decode step has added a token to each sequence: the bounds of the page that it fell into, where latency counts
        dict(name="bounds_append", op="bounds", qtype="q4_0", batch=16, nq=1, heads=32, kv_heads=8, d=128, length=4096, spread=4000, page=64, new=1),
        # the bounds of a whole context once its prompt is in the cache
        dict(name="bounds_context_q4_1", op="bounds", qtype="q4_1", batch=2, nq=1, heads=16, kv_heads=4, d=128, length=65536, spread=9000, page=64, new=0),
        # the pages that single tokens of many sequences of uneven lengths read next, one sequence empty
        dict(name="select_batch", op="select", qtype="q4_0", batch=32, nq=1, heads=32, kv_heads=8, d=128, length=16384, spread=15000, page=64, share=1, keep=32, sink=1, recent=2, causal=False, window=0),
        # one token of one very long sequence in small pages: 16384 scores a head
        dict(name="select_long_q8", op="select", qtype="q8_0", batch=1, nq=1, heads=16, kv_heads=2, d=64, length=524288, spread=0, page=32, share=1, keep=256, sink=1, recent=4, causal=False, window=0),
        # one query of one sequence, a head for each query head: choice and attention where latency counts
        dict(name="sparse_short", op="sparse", qtype="q4_0", batch=1, nq=1, heads=8, kv_heads=8, d=64, length=4801, spread=0, page=16, share=1, keep=24, sink=1, recent=2, causal=False, window=0),
        # single tokens of many sequences, grouped heads, an eighth of the longest ones read
        dict(name="sparse_batch", op="sparse", qtype="q4_0", batch=32, nq=1, heads=32, kv_heads=8, d=128, length=16384, spread=15000, page=64, share=1, keep=32, sink=1, recent=2, causal=False, window=0),
        # every token of a 64 x 64 map over a full memory bank (7 maps and 64 pointer tokens), 16 neighbouring tokens a choice
        dict(name="sparse_track", op="sparse", qtype="q8_0", batch=1, nq=4096, heads=1, kv_heads=1, d=256, length=28736, spread=0, page=64, share=16, keep=64, sink=0, recent=1, causal=False, window=0),
        # a few drafted tokens at once, causal, each with its own choice, pages that end inside a step
        dict(name="sparse_draft_q4_1", op="sparse", qtype="q4_1", batch=5, nq=5, heads=12, kv_heads=4, d=128, length=30011, spread=20000, page=48, share=1, keep=40, sink=2, recent=2, causal=True, window=0),
        # what single tokens of many sequences add to the weights of their caches
        dict(name="weights_decode", op="weights", qtype="q4_0", batch=32, nq=1, heads=32, kv_heads=8, d=128, length=16384, spread=15000, page=64, causal=False, window=0, decay=0.95),
        # the weights that one frame's 64 x 64 queries give to a memory bank's tokens
        dict(name="weights_track", op="weights", qtype="q4_0", batch=1, nq=4096, heads=1, kv_heads=1, d=256, length=28736, spread=0, page=64, causal=False, window=0, decay=1.0),
        # a quarter of the tokens of many sequences kept, some sequences shorter than that
        dict(name="evict_batch", op="evict", qtype="q4_0", batch=8, nq=1, heads=32, kv_heads=8, d=128, length=16384, spread=15000, page=64, keep=4096, sink=4, recent=64),
        # one very long sequence, an eighth of it kept
        dict(name="evict_long_q8", op="evict", qtype="q8_0", batch=1, nq=1, heads=16, kv_heads=2, d=64, length=524288, spread=0, page=32, keep=65536, sink=16, recent=1024),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = [work(c) for c in listed()]
    most = {k: max(w[k] for w in most) for k in ("bytes", "flops")}
    while True:
        op = rng.choice(["bounds", "select", "sparse", "sparse", "weights", "weights", "evict"])
        kv = _log(rng, 1, 16)
        length = _log(rng, 1, 524288)
        c = dict(op=op, qtype=rng.choice(sorted(QTYPES)), batch=_log(rng, 1, 32), nq=1, heads=kv * rng.choice([1, 2, 3, 4, 8]), kv_heads=kv,
                 d=rng.choice([64, 128, 256]), length=length, spread=rng.choice([0, int(length * rng.random())]), page=16 * _log(rng, 1, 16))
        if op == "bounds":
            c["new"] = rng.choice([0, _log(rng, 1, 4096)])
        if op in ("select", "sparse"):
            group = c["heads"] // kv
            c["share"] = rng.choice([1, 1 + rng.randrange((16 if c["d"] == 256 else 32) // group)])
            c["keep"] = _log(rng, 4, 256)
            c["sink"], c["recent"] = rng.randrange(3), rng.randrange(3)
        if op in ("select", "sparse", "weights"):
            c["nq"] = rng.choice([1, _log(rng, 1, 16), _log(rng, 16, 4096)])
            c["causal"] = rng.random() < 0.6
            c["window"] = _log(rng, 64, 16384) if c["causal"] and rng.random() < 0.3 else 0
        if op == "weights":
            c["decay"] = rng.choice([1.0, 0.95])
        if op == "evict":
            c["keep"] = min(length, _log(rng, 1, 65536))
            c["sink"], c["recent"] = rng.randrange(1 + c["keep"] // 4), rng.randrange(1 + c["keep"] // 4)
        # what the plain form holds in 32 bits: the unpacked rows; scores of every page; the chosen rows; scores of every token
        pages = -(-length // c["page"])
        blocks = -(-c["nq"] // c.get("share", 1))
        if c["batch"] * kv * length * c["d"] > 1.2e9:
            continue
        if op in ("select", "sparse") and c["batch"] * c["heads"] * c["nq"] * pages > 3e8:
            continue
        if op == "sparse" and c["batch"] * blocks * kv * min(c["keep"], pages) * c["page"] * c["d"] > 3e8:
            continue
        if op == "weights" and c["batch"] * c["heads"] * c["nq"] * length > 6e8:
            continue
        w = work(c)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"]:
            return c


def _lengths(case):
    """Token count of each sequence: from `length` down by up to `spread`, the last of several of them empty."""
    b, length, spread = case["batch"], case["length"], case["spread"]
    out = [length - (i * 7919 * max(spread // 9, 1)) % (spread + 1) for i in range(b)]
    if b > 8 and spread:
        out[-1] = 0
    return out


def _row_bytes(case):
    d, t = case["d"], case["qtype"]
    return {"q4_0": d // 2 + d // 16, "q4_1": d // 2 + d // 8, "q8_0": d + d // 16}[t]


def _range(case, n, i):
    """Positions [lo, hi) that query i sees in a sequence of n tokens."""
    if not case["causal"]:
        return 0, n
    hi = n - case["nq"] + i + 1
    lo = max(0, hi - case["window"]) if case["window"] else 0
    return lo, max(hi, 0)


def _page_range(case, n, first, last):
    """Pages [a, b) that queries first .. last see between them."""
    lo, hi = _range(case, n, first)[0], _range(case, n, last)[1]
    return lo // case["page"], max(lo // case["page"], -(-hi // case["page"]))


def work(case):
    d, row, kv, page, nq = case["d"], _row_bytes(case), case["kv_heads"], case["page"], case["nq"]
    op, heads = case["op"], case["heads"]
    group = heads // kv
    lengths = _lengths(case)
    if op == "bounds":
        touched = sum(-(-n // page) - (max(0, n - case["new"]) // page if case["new"] else 0) for n in lengths)
        tokens = sum(n - (max(0, n - case["new"]) // page * page if case["new"] else 0) for n in lengths)
        # bounds are written, and returned as the values that they stand for
        return {"bytes": kv * (tokens * row + touched * (2 * d + 4 + 8 * d)), "flops": 2 * kv * tokens * d}
    if op in ("select", "sparse"):
        share, keep = case["share"], case["keep"]
        moved = 2 * case["batch"] * nq * heads * d + 4 * case["batch"] * kv * -(-nq // share) * keep
        flops = 0
        for n in lengths:
            spans = [_page_range(case, n, f, min(nq, f + share) - 1) for f in range(0, nq, share)]
            sees = [b - a for a, b in spans]
            union = max(b for _, b in spans) - min(a for a, _ in spans)
            moved += kv * union * (2 * d + 4)
            flops += 2 * d * group * kv * sum(s * min(share, nq - i * share) for i, s in enumerate(sees))
            if op == "select":
                moved += 4 * kv * len(spans) * -(-case["length"] // page)
            else:
                chosen = [min(s, keep) * page for s in sees]
                moved += kv * 2 * row * min(union * page, sum(chosen)) + 4 * nq * heads
                flops += 4 * d * heads * sum(s * min(share, nq - i * share) for i, s in enumerate(chosen))
        if op == "sparse":
            moved += 2 * case["batch"] * nq * heads * d
        return {"bytes": moved, "flops": flops}
    if op == "weights":
        seen = pairs = 0
        for n in lengths:
            first, last = _range(case, n, 0)[0], _range(case, n, nq - 1)[1]
            seen += max(0, last - first)
            if case["causal"] and nq * n:
                pairs += sum(max(0, hi - lo) for lo, hi in (_range(case, n, i) for i in range(nq)))
            else:
                pairs += nq * n
        moved = kv * seen * row + 8 * kv * sum(lengths) + case["batch"] * nq * heads * (2 * d + 4)
        return {"bytes": moved, "flops": 2 * d * heads * pairs}
    kept = sum(min(n, case["keep"]) for n in lengths)
    # weights; rows out of their pages, into others; what is returned: positions, weights and the rows as f16
    return {"bytes": kv * (4 * sum(lengths) + kept * (4 * row + 8 + 4 * d)), "flops": 2 * kv * kept * d}


# ------------------------------------------------------------------------------------------------ inputs
def _inputs(case, seed):
    """The tensors of a case, from the seed alone. Keys have channels of uneven size and offset, and drift over the tokens, as
    those of a text or a stream of frames do."""
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    d, kv, batch, nq = case["d"], case["kv_heads"], case["batch"], case["nq"]
    per = -(-case["length"] // case["page"])
    extra = -(-min(case["keep"], case["length"]) // case["page"]) if case["op"] == "evict" else 0
    total = batch * (per + extra)

    def rand(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    pool = torch.randperm(total, device=dev, generator=g).to(torch.int32)
    lengths = torch.tensor(_lengths(case), dtype=torch.int32, device=dev)
    x = dict(pages=pool[:batch * per].view(batch, per), pages_out=pool[batch * per:].view(batch, extra), lengths=lengths)
    n = total * case["page"]
    k = rand(n, kv, d).mul_(torch.exp(0.4 * rand(1, kv, d))).add_(0.7 * rand(1, kv, d))
    k.view(total, case["page"], kv, d).add_(0.5 * rand(total, 1, kv, d))  # tokens of a page are alike
    v = rand(n, kv, d).mul_(torch.exp(0.4 * rand(1, kv, 1)))
    x["k"], x["v"] = k.half(), v.half()
    x["q"] = (0.8 * rand(batch, nq, case["heads"], d)).half()
    if case["op"] in ("weights", "evict"):
        # gathered weights span orders of magnitude; the newest tokens of all and some old ones have none yet
        w = torch.exp(2.0 * rand(batch, kv, per * case["page"]))
        x["weights"] = torch.where(rand(batch, kv, per * case["page"]) > 1.5, 0.0, w)
    return x


_engine = []


def _framework():
    """This repository's package and one engine that works on torch's stream."""
    import __graft_entry__
    s3b = __graft_entry__._pkg()
    if not _engine:
        _engine.append(s3b.Engine(0))
        _engine[0].set_stream(torch.cuda.current_stream().cuda_stream)
    return s3b, _engine[0]


def prepare(case, seed):
    x = _inputs(case, seed)
    op, kv, d, page, batch = case["op"], case["kv_heads"], case["d"], case["page"], case["batch"]
    n_slots = x["k"].shape[0]
    state = {"case": case, "scale": d ** -0.5, "pages": x["pages"], "lengths": x["lengths"], "q": x["q"]}
    every = torch.arange(n_slots, device="cuda")
    plain = None if own and op != "weights" else [_quantise(case["qtype"], x[n]) for n in "kv"]
    if op == "weights":  # what the attention before it has given
        state["lse"] = _lse(case, plain[0], x)
        state["weights"] = x["weights"]
    # the cache that a program holds: the framework's own, or plain tensors of codes, scales and minima
    if own:
        s3b, eng = _framework()
        state["engine"] = eng
        state["cache"] = s3b.KVCache(QTYPES[case["qtype"]], n_slots // page, page, kv, d)
        eng.cache_write(state["cache"], x["k"], x["v"], every)
    else:
        state["cache"] = plain
    if op in ("bounds", "select", "sparse"):
        if own:
            state["bounds"] = s3b.KVBounds(state["cache"])
            eng.cache_bounds(state["cache"], state["bounds"], x["pages"], x["lengths"])
        else:
            state["bounds"] = [torch.zeros(n_slots // page, kv, 2, d, dtype=torch.int8, device="cuda"),
                               torch.zeros(n_slots // page, kv, device="cuda")]
            _bounds(state, 0)
    if op == "bounds":  # the pages that hold the newest tokens
        last = [-(-n // page) for n in _lengths(case)]
        first = [max(0, n - case["new"]) // page if case["new"] else 0 for n in _lengths(case)]
        which = [(b, j) for b in range(batch) for j in range(first[b], last[b])]
        at = torch.tensor(which, dtype=torch.int64, device="cuda").view(-1, 2)
        state["touched"] = x["pages"][at[:, 0], at[:, 1]].long()
    if op in ("select", "sparse"):
        blocks = -(-case["nq"] // case["share"])
        state["selected"] = torch.empty(batch, blocks, kv, case["keep"], dtype=torch.int32, device="cuda")
        if op == "select":
            state["scores"] = torch.empty(batch, blocks, kv, x["pages"].shape[1], device="cuda")
        else:
            state["out"] = torch.empty_like(x["q"])
            state["lse"] = torch.empty(batch, case["nq"], case["heads"], device="cuda")
    if op == "evict":
        state["weights"], state["pages_out"] = x["weights"], x["pages_out"]
        kept = min(case["keep"], case["length"])
        state["lengths_out"] = torch.empty_like(x["lengths"])
        state["kept"] = torch.empty(batch, kv, kept, dtype=torch.int32, device="cuda")
        state["weights_out"] = torch.empty(batch, kv, kept, device="cuda")
        at = torch.arange(kept, device="cuda")
        slots = x["pages_out"].long()[:, at // page] * page + at % page
        state["slots_out"] = torch.where(at < x["lengths"][:, None], slots, -1).flatten()
        state["k_out"], state["v_out"] = (torch.empty(batch * kept, kv, d, dtype=torch.float16, device="cuda") for _ in "kv")
    torch.cuda.synchronize()
    return state


# ------------------------------------------------------------------------------------------------ plain form
def _over(x, by):
    """x / by rounded once: the division by a number multiplies by its rounded reciprocal on the GPU."""
    return x / torch.full_like(x, by)


def _under(by, x):
    return torch.full_like(x, by) / x


def _quantise(qtype, rows):
    """Codes, scale (and minimum) of rows [n, heads, d], in the formats' own float32 steps."""
    x = torch.nan_to_num(rows.float(), nan=0.0, posinf=LIMIT, neginf=-LIMIT).clamp(-LIMIT, LIMIT)
    x = x.unflatten(-1, (-1, 32))
    if qtype == "q4_1":
        low = x.amin(-1, keepdim=True)
        scale = _over(x.amax(-1, keepdim=True) - low, 15.0)
        inv = torch.where(scale != 0, 1.0 / scale, 0.0)
        return [((x - low) * inv + 0.5).clamp(0, 15).to(torch.uint8), scale.half(), low.half()]
    size = x.abs()
    peak = size.amax(-1, keepdim=True)
    if qtype == "q8_0":
        scale = _over(peak, 127.0)
        inv = torch.where(scale != 0, 1.0 / scale, 0.0)
        y = x * inv
        whole = y.trunc()
        return [(whole + torch.where((y - whole).abs() >= 0.5, y.sign(), 0.0)).to(torch.int8), scale.half()]
    # q4_0 scales by the value of largest magnitude with its sign, the first of equals
    place = torch.arange(32, device=x.device).expand_as(x)
    first = torch.where(size == peak, place, 32).amin(-1, keepdim=True)
    scale = torch.where(place == first, x, 0.0).sum(-1, keepdim=True) / -8.0
    inv = torch.where(scale != 0, 1.0 / scale, 0.0)
    return [(x * inv + 8.5).clamp(0, 15).to(torch.uint8), scale.half()]


def _values(qtype, codes, scale, low=None):
    """Rows in 32 bits of codes [..., blocks, 32] and scales (and minima) [..., blocks, 1]."""
    x = (codes.float() - 8.0) * scale.float() if qtype == "q4_0" else codes.float() * scale.float()
    if low is not None:
        x = x + low.float()
    return x.flatten(-2)


def _all_slots(state):
    """Slots [batch, max tokens] of the tokens of each sequence, in order."""
    page = state["case"]["page"]
    return (state["pages"].long()[:, :, None] * page + torch.arange(page, device="cuda")).flatten(1)


def _spans(case, lengths):
    """Positions [lo, hi) that each query sees: two tensors [batch, nq]."""
    n = lengths.long()[:, None].expand(-1, case["nq"])
    if not case["causal"]:
        return torch.zeros_like(n), n
    hi = n - case["nq"] + torch.arange(1, case["nq"] + 1, device="cuda")
    lo = hi - case["window"] if case["window"] else torch.zeros_like(hi)
    return lo.clamp(min=0), hi.clamp(min=0)


def _grouped(case, q):
    """q [batch, nq, heads, d] as f32 [batch, kv heads, group, nq, d]."""
    return q.float().unflatten(2, (case["kv_heads"], -1)).permute(0, 2, 3, 1, 4)


def _lse(case, keys, x):
    """ln sum exp(scale q k) of every row over the tokens that it sees, [batch, nq, heads]."""
    s = _scores(case, keys, {"case": case, **x})
    return torch.logsumexp(s, -1).permute(0, 3, 1, 2).flatten(2).contiguous()


def _scores(case, keys, state):
    """scale q k of every row over all tokens, -inf where it does not see them: [batch, kv heads, group, nq, tokens]."""
    slots = _all_slots(state)
    k = _values(case["qtype"], *(t[slots] for t in keys)).permute(0, 2, 3, 1)     # [batch, kv heads, d, tokens]
    s = torch.matmul(_grouped(case, state["q"]).flatten(2, 3), k) * case["d"] ** -0.5
    lo, hi = _spans(case, state["lengths"])
    at = torch.arange(slots.shape[1], device="cuda")
    hidden = (at < lo[..., None]) | (at >= hi[..., None])
    return s.unflatten(2, (-1, case["nq"])).masked_fill_(hidden[:, None, None], -math.inf)


def _bounds(state, new):
    """Writes the bounds of the pages that hold the last `new` tokens of each sequence (0: of all its pages)."""
    case, (codes, steps) = state["case"], state["bounds"]
    page, pages, n = case["page"], state["pages"].long(), state["lengths"].long()[:, None]
    first = torch.clamp(n - new, min=0) // page if new else torch.zeros_like(n)
    many = min(pages.shape[1], (new + page - 2) // page + 1) if new else pages.shape[1]
    j = first + torch.arange(many, device="cuda")                                # [batch, pages looked at]
    used = j * page < n
    which = pages.gather(1, j.clamp(max=pages.shape[1] - 1))[used]
    at = torch.arange(page, device="cuda")
    there = (j[used][:, None] * page + at < n.expand_as(j)[used][:, None])[..., None, None]
    k = _values(case["qtype"], *(t[which[:, None] * page + at] for t in state["cache"][0])).half().float()
    low = torch.where(there, k, math.inf).amin(1)                                  # [pages, heads, d]
    high = torch.where(there, k, -math.inf).amax(1)
    peak = torch.maximum(low.abs(), high.abs()).amax(-1, keepdim=True)
    inv = torch.where(peak != 0, _under(127.0, peak), 0.0)
    codes[which] = torch.stack([(low * inv).floor().clamp(min=-127), (high * inv).ceil().clamp(max=127)], -2).to(torch.int8)
    steps[which] = _over(peak, 127.0).squeeze(-1)


def _select(state):
    case, (codes, steps) = state["case"], state["bounds"]
    page, nq, share, keep = case["page"], case["nq"], case["share"], case["keep"]
    pages = state["pages"].long()
    x = torch.nan_to_num(_grouped(case, state["q"]), nan=0.0, posinf=65504.0, neginf=-65504.0)
    peak = x.abs().amax(-1, keepdim=True)
    t = _over(peak, 127.0)
    c = (x * torch.where(peak != 0, _under(127.0, peak), 0.0)).round().clamp(-127, 127).flatten(2, 3)
    low, high = (codes[pages][..., e, :].permute(0, 2, 3, 1).float() for e in (0, 1))  # [batch, kv heads, d, pages]
    dot = torch.matmul(c.clamp(min=0), high) + torch.matmul(c.clamp(max=0), low)    # whole numbers below 2^24
    s = (dot * steps[pages].permute(0, 2, 1)[:, :, None]) * t.flatten(2, 3)
    s = s.unflatten(2, (-1, nq)).amax(2)                                            # [batch, kv heads, nq, pages]
    blocks = -(-nq // share)
    s = torch.nn.functional.pad(s, (0, 0, 0, blocks * share - nq), value=-math.inf).unflatten(2, (blocks, share)).amax(3)
    lo, hi = _spans(case, state["lengths"])
    lo, hi = lo[:, ::share], hi[:, torch.arange(share - 1, blocks * share, share, device="cuda").clamp(max=nq - 1)]
    a, b = (lo // page)[:, None, :, None], ((hi + page - 1) // page)[:, None, :, None]
    j = torch.arange(pages.shape[1], device="cuda")
    s = torch.where((j >= a) & (j < b), s, -math.inf)
    forced = (s > -math.inf) & ((j < a + case["sink"]) | (j >= b - case["recent"]))
    order = torch.argsort(torch.where(forced, math.inf, s), dim=-1, descending=True, stable=True)[..., :keep]
    chosen = torch.where(s.gather(-1, order) > -math.inf, order, pages.shape[1]).sort(-1).values
    chosen = torch.where(chosen < pages.shape[1], chosen, -1)
    chosen = torch.nn.functional.pad(chosen, (0, keep - chosen.shape[-1]), value=-1)
    return chosen.transpose(1, 2).to(torch.int32).contiguous(), s.transpose(1, 2).contiguous()


def _attend(state, selected):
    case, q = state["case"], state["q"]
    page, nq, share, kv, d = case["page"], case["nq"], case["share"], case["kv_heads"], case["d"]
    blocks, group = selected.shape[1], case["heads"] // kv
    batch = selected.shape[0]
    chosen = selected[..., :state["pages"].shape[1]].long()
    where = state["pages"].long()[torch.arange(batch, device="cuda")[:, None, None, None], chosen.clamp(min=0)]
    at = torch.arange(page, device="cuda")
    slots = (where[..., None] * page + at).flatten(3)                               # [batch, blocks, kv heads, tokens]
    token = torch.where(chosen[..., None] >= 0, chosen[..., None] * page + at, -1).flatten(3)
    head = torch.arange(kv, device="cuda")[:, None]
    k, v = (_values(case["qtype"], *(t[slots, head] for t in part)) for part in state["cache"])
    x = torch.nn.functional.pad(q.float(), (0, 0, 0, 0, 0, blocks * share - nq))
    x = x.view(batch, blocks, share, kv, group, d).permute(0, 1, 3, 2, 4, 5).flatten(3, 4)  # [batch, blocks, kv heads, rows, d]
    s = torch.matmul(x, k.transpose(-1, -2)) * state["scale"]
    lo, hi = (torch.nn.functional.pad(t, (0, blocks * share - nq)).view(batch, blocks, 1, share, 1, 1) for t in _spans(case, state["lengths"]))
    token = token[:, :, :, None, None]
    seen = ((token >= lo) & (token < hi) & (token >= 0)).expand(-1, -1, -1, -1, group, -1).flatten(3, 4)
    s = torch.where(seen, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    lse = (top + torch.log(total)).view(batch, blocks, kv, share, group).permute(0, 1, 3, 2, 4).reshape(batch, blocks * share, kv * group)
    o = o.view(batch, blocks, kv, share, group, d).permute(0, 1, 3, 2, 4, 5).reshape(batch, blocks * share, kv * group, d)
    return o[:, :nq].half(), lse[:, :nq].contiguous()


def _weights(state):
    case = state["case"]
    s = _scores(case, state["cache"][0], state)                                     # [batch, kv heads, group, nq, tokens]
    lse = state["lse"].unflatten(2, (case["kv_heads"], -1)).permute(0, 2, 3, 1)[..., None]
    p = torch.where(s > -math.inf, torch.exp(s - lse), 0.0)
    there = torch.arange(s.shape[-1], device="cuda") < state["lengths"][:, None, None]
    w = state["weights"]
    w.copy_(torch.where(there, case["decay"] * w + p.sum((2, 3)), w))
    return w


def _evict(state):
    case = state["case"]
    n, keep = state["lengths"].long()[:, None, None], state["kept"].shape[-1]
    page = case["page"]
    w = state["weights"]
    at = torch.arange(w.shape[-1], device="cuda")
    there = at < n
    w = torch.where(there, w, -math.inf)
    forced = there & ((at < case["sink"]) | (at >= n - case["recent"]))
    order = torch.argsort(torch.where(forced, math.inf, w), dim=-1, descending=True, stable=True)[..., :keep]
    order = torch.where(order < n, order, w.shape[-1]).sort(-1).values
    valid = order < w.shape[-1]
    kept = torch.where(valid, order, -1)
    weights = torch.where(valid, state["weights"].gather(-1, kept.clamp(min=0)), 0.0)
    # [batch, kept] slots of the rows' new places, [batch, kept, heads] of their old ones
    new = torch.arange(keep, device="cuda")
    to = state["pages_out"].long()[:, new // page] * page + new % page
    which = valid[:, 0]
    source = _all_slots(state)[torch.arange(len(to), device="cuda")[:, None, None], kept.clamp(min=0)].transpose(1, 2)[which]
    head = torch.arange(case["kv_heads"], device="cuda")
    to = to[which]
    state["cache"] = [[t.index_put_((to,), t[source, head]) for t in part] for part in state["cache"]]
    slots = state["slots_out"]
    rows = [torch.where((slots >= 0)[:, None, None], _values(case["qtype"], *(t[slots.clamp(min=0)] for t in part)), 0.0).half()
            for part in state["cache"]]
    return kept.to(torch.int32), weights, state["lengths"].clamp(max=keep), *rows


def run(state):
    case, op = state["case"], state["case"]["op"]
    if own:
        eng, cache = state["engine"], state["cache"]
        if op == "bounds":
            eng.cache_bounds(cache, state["bounds"], state["pages"], state["lengths"], new=case["new"] or None)
            return state["bounds"].values(state["touched"])
        if op == "select":
            eng.cache_select(state["bounds"], state["q"], state["selected"], state["pages"], state["lengths"], share=case["share"],
                             sink=case["sink"], recent=case["recent"], causal=case["causal"], window=case["window"], scores=state["scores"])
            return state["selected"], state["scores"]
        if op == "sparse":
            eng.cache_select(state["bounds"], state["q"], state["selected"], state["pages"], state["lengths"], share=case["share"],
                             sink=case["sink"], recent=case["recent"], causal=case["causal"], window=case["window"])
            eng.cache_attention_selected(cache, state["q"], state["out"], state["selected"], state["pages"], state["lengths"], state["scale"],
                                         share=case["share"], causal=case["causal"], window=case["window"], lse=state["lse"])
            return state["selected"], state["out"], state["lse"]
        if op == "weights":
            eng.cache_weights(cache, state["q"], state["lse"], state["weights"], state["pages"], state["lengths"], state["scale"],
                              decay=case["decay"], causal=case["causal"], window=case["window"])
            return state["weights"]
        eng.cache_evict(cache, state["weights"], state["pages"], state["lengths"], state["pages_out"], state["lengths_out"], state["kept"],
                        sink=case["sink"], recent=case["recent"], weights_out=state["weights_out"])
        eng.cache_read(cache, state["slots_out"], state["k_out"], state["v_out"])
        return state["kept"], state["weights_out"], state["lengths_out"], state["k_out"], state["v_out"]
    if op == "bounds":
        _bounds(state, case["new"])
        codes, steps = (t[state["touched"]] for t in state["bounds"])
        return codes * steps[..., None, None]
    if op == "select":
        return _select(state)
    if op == "sparse":
        selected, _ = _select(state)
        return selected, *_attend(state, selected)
    if op == "weights":
        return _weights(state)
    return _evict(state)


# ------------------------------------------------------------------------------------------------ 64 bits
def _f32(t):
    """A 32-bit step of a definition: the value in 64 bits, rounded."""
    return t.float().double()


def _held(qtype, rows):
    """The values that rows [..., d] stand for once quantised, in 64 bits. The formats define their codes by float32
    steps, so each of those steps is taken exactly in 64 bits and then rounded to 32."""
    x = rows.double().reshape(-1, 32)
    if qtype == "q4_1":
        low, high = x.min(1, keepdim=True).values, x.max(1, keepdim=True).values
        step = _f32(_f32(high - low) / 15)
    elif qtype == "q8_0":
        step = _f32(x.abs().max(1, keepdim=True).values / 127)
    else:
        order = x.abs().sort(dim=1, descending=True, stable=True).indices[:, :1]
        step = x.gather(1, order) / -8
    inv = torch.zeros_like(step)
    inv[step != 0] = _f32(1 / step[step != 0])
    kept = step.half().double()
    if qtype == "q4_1":
        code = _f32(_f32(_f32(x - low) * inv) + 0.5).floor().clamp(max=15)
        y = code * kept + low.half().double()
    elif qtype == "q8_0":
        y = _f32(x * inv)
        y = torch.copysign((y.abs() + 0.5).floor(), y) * kept
    else:
        y = (_f32(_f32(x * inv) + 8.5).floor().clamp(max=15) - 8) * kept
    return y.view(rows.shape)


def _tokens(case, x, b, n):
    """Slots of the first n tokens of sequence b."""
    page = case["page"]
    return (x["pages"][b].long()[:, None] * page + torch.arange(page, device="cuda")).flatten()[:n]


def _page_bounds(keys, page):
    """Codes and steps of the bounds of the pages of one head's keys [tokens, d], in 64 bits."""
    keys = keys.half().double()
    pages = torch.cat([keys, keys[-1:].expand(-len(keys) % page, -1)]).view(-1, page, keys.shape[1])
    low, high = pages.min(1).values, pages.max(1).values
    peak = torch.cat([low, high], 1).abs().max(1, keepdim=True).values
    inv = torch.zeros_like(peak)
    inv[peak > 0] = _f32(127 / peak[peak > 0])
    return (_f32(low * inv).floor().clamp(min=-127), _f32(high * inv).ceil().clamp(max=127)), _f32(peak / 127)


def _row_scores(q, bounds, step):
    """Scores [rows, pages] of queries [rows, d]."""
    peak = q.abs().max(1, keepdim=True).values
    inv = torch.zeros_like(peak)
    inv[peak > 0] = _f32(127 / peak[peak > 0])
    c = _f32(q * inv).round().clamp(-127, 127)
    dot = torch.where(c > 0, c, 0.0) @ bounds[1].T + torch.where(c < 0, c, 0.0) @ bounds[0].T
    return _f32(_f32(dot * step.T) * _f32(peak / 127))


def exact(case, seed):
    x = _inputs(case, seed)
    op, qtype, page, nq, kv, d = case["op"], case["qtype"], case["page"], case["nq"], case["kv_heads"], case["d"]
    group, lengths = case["heads"] // kv, _lengths(case)
    dev = "cuda"
    if op == "bounds":
        got = []
        for b, n in enumerate(lengths):
            first = max(0, n - case["new"]) // page if case["new"] else 0
            if first * page < n:
                keys = _held(qtype, x["k"][_tokens(case, x, b, n)[first * page:]])
                heads = [_page_bounds(keys[:, h], page) for h in range(kv)]
                got.append(torch.stack([torch.stack(c, 1) * step[:, None] for c, step in heads], 1))
        return torch.cat(got) if got else torch.zeros(0, kv, 2, d, dtype=torch.float64, device=dev)
    if op in ("select", "sparse"):
        share, keep = case["share"], case["keep"]
        blocks, most = -(-nq // share), x["pages"].shape[1]
        if case["batch"] * kv * blocks > 4096:
            return None
        selected = torch.full((case["batch"], blocks, kv, keep), -1, dtype=torch.int32, device=dev)
        scores = torch.full((case["batch"], blocks, kv, most), -math.inf, dtype=torch.float64, device=dev)
        out = torch.zeros(x["q"].shape, dtype=torch.float64, device=dev)
        lse = torch.full(x["q"].shape[:3], -math.inf, dtype=torch.float64, device=dev)
        for b, n in enumerate(lengths):
            if not n:
                continue
            slots = _tokens(case, x, b, n)
            for h in range(kv):
                keys, values = _held(qtype, x["k"][slots, h]), _held(qtype, x["v"][slots, h])
                bounds, step = _page_bounds(keys, page)
                for i in range(blocks):
                    rows = range(i * share, min(nq, (i + 1) * share))
                    a, e = _page_range(case, n, rows[0], rows[-1])
                    if a >= e:
                        continue
                    q = x["q"][b, rows[0]:rows[-1] + 1, h * group:(h + 1) * group].double().reshape(-1, d)
                    s = _row_scores(q, bounds, step).max(0).values[a:e]
                    scores[b, i, h, a:e] = s
                    if e - a <= keep:
                        chosen = torch.arange(a, e, device=dev)
                    else:
                        middle = s[case["sink"]:e - a - case["recent"]]
                        best = middle.sort(descending=True, stable=True).indices[:keep - case["sink"] - case["recent"]]
                        ends = torch.tensor([*range(a, a + case["sink"]), *range(e - case["recent"], e)], dtype=torch.int64, device=dev)
                        chosen = torch.cat([ends, best + a + case["sink"]]).sort().values
                    selected[b, i, h, :len(chosen)] = chosen.int()
                    if op == "sparse":
                        token = (chosen[:, None] * page + torch.arange(page, device=dev)).flatten()
                        token = token[token < n]
                        span = torch.tensor([_range(case, n, r) for r in rows], device=dev).repeat_interleave(group, 0)
                        z = (q @ keys[token].T) * d ** -0.5
                        z[(token < span[:, :1]) | (token >= span[:, 1:])] = -math.inf
                        o = z.softmax(-1).nan_to_num(0.0) @ values[token]
                        out[b, rows[0]:rows[-1] + 1, h * group:(h + 1) * group] = o.view(len(rows), group, d)
                        lse[b, rows[0]:rows[-1] + 1, h * group:(h + 1) * group] = z.logsumexp(-1).view(len(rows), group)
        return (selected, scores) if op == "select" else (selected, out, lse)
    if op == "weights":
        lse = _lse(case, _quantise(qtype, x["k"]), x).double()
        w = x["weights"].double()
        for b, n in enumerate(lengths):
            if not n:
                continue
            slots, at = _tokens(case, x, b, n), torch.arange(n, device=dev)
            w[b, :, :n] *= case["decay"]
            spans = torch.tensor([_range(case, n, i) for i in range(nq)], device=dev)
            for h in range(kv):
                k = _held(qtype, x["k"][slots, h])
                for first in range(0, nq, 1024):
                    rows = slice(first, min(nq, first + 1024))
                    hide = (at < spans[rows, :1]) | (at >= spans[rows, 1:])
                    for m in range(h * group, (h + 1) * group):
                        s = (x["q"][b, rows, m].double() @ k.T) * d ** -0.5
                        w[b, h, :n] += torch.exp(s - lse[b, rows, m, None]).masked_fill(hide, 0.0).sum(0)
        return w
    keep = min(case["keep"], case["length"])
    kept = torch.full((case["batch"], kv, keep), -1, dtype=torch.int32, device=dev)
    weights = torch.zeros(case["batch"], kv, keep, dtype=torch.float64, device=dev)
    rows = [torch.zeros(case["batch"], keep, kv, d, dtype=torch.float64, device=dev) for _ in "kv"]
    for b, n in enumerate(lengths):
        m = min(n, keep)
        if not n:
            continue
        slots = _tokens(case, x, b, n)
        for h in range(kv):
            w = x["weights"][b, h, :n].double()
            if n <= keep:
                chosen = torch.arange(n, device=dev)
            else:
                sink, end = case["sink"], n - case["recent"]
                best = w[sink:end].sort(descending=True, stable=True).indices[:keep - sink - case["recent"]] + sink
                chosen = torch.cat([torch.arange(sink, device=dev), best, torch.arange(end, n, device=dev)]).sort().values
            kept[b, h, :m] = chosen.int()
            weights[b, h, :m] = w[chosen]
            for r, name in zip(rows, "kv"):
                r[b, :m, h] = _held(qtype, x[name][slots[chosen], h])
    return kept, weights, torch.tensor(lengths, dtype=torch.int32, device=dev).clamp(max=keep), *(r.flatten(0, 1) for r in rows)
