"""Cases of the key/value cache operators: quantising tokens as they are written, reading them back, and
attention over the quantised cache.

A cache holds, for every token slot and key/value head, one key row and one value row of d values in blocks of
32, in one of the block formats of the .ggml files:

  q4_0  codes 0..15, value (code - 8) * scale
  q4_1  codes 0..15, value code * scale + minimum
  q8_0  codes -127..127, value code * scale

with scale and minimum held as float16. Attention takes the pages of each sequence from a page table and softmaxes
over the first lengths[b] tokens: out = softmax(scale * q k^T) v, query head h reading key/value head
h // (heads / kv_heads). With `causal` query i of nq is the token at position length - nq + i and sees no later
position; with `window` > 0 it sees only the last `window` positions up to its own. A row that sees nothing is zero.
"""
import math

import torch

own = False

QTYPES = {"q4_0": 2, "q4_1": 3, "q8_0": 8}
DTYPES = {"f16": torch.float16, "f32": torch.float32}
LIMIT = 65024.0  # magnitude that a value is held to before it is quantised


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the pointer tokens that one object adds to its memory per frame: four rows, where latency counts
        dict(name="write_pointers", op="write", qtype="q4_0", n=4, heads=1, d=256, page=16, slots=64, order="pages", src="f32", dst="f16"),
        # one frame's 64 x 64 memory map, projected to keys and values of the memory attention's single head
        dict(name="write_frame", op="write", qtype="q4_0", n=4096, heads=1, d=256, page=64, slots=28736, order="pages", src="f16", dst="f16"),
        # a long prompt with an odd count, kept in 8 bits and read back in full precision
        dict(name="write_prompt_q8", op="write", qtype="q8_0", n=20011, heads=4, d=64, page=32, slots=20032, order="pages", src="f32", dst="f32"),
        # the largest fill: a whole context of grouped heads
        dict(name="write_context_q4_1", op="write", qtype="q4_1", n=65536, heads=4, d=128, page=64, slots=65536, order="pages", src="f16", dst="f16"),
        # a full memory bank (7 maps of 64 x 64 and 64 pointer tokens) read back as keys and values
        dict(name="read_bank", op="read", qtype="q4_0", n=28736, heads=1, d=256, page=64, slots=28736, order="pages", skip=0, dst="f16"),
        # scattered tokens of an 8-bit cache, an odd head count, some rows of the list switched off
        dict(name="read_scattered_q8", op="read", qtype="q8_0", n=5003, heads=5, d=128, page=16, slots=16384, order="any", skip=7, dst="f32"),
        # one query of one short sequence, a head for each query head: latency
        dict(name="decode_short", op="attend", qtype="q4_0", batch=1, nq=1, heads=8, kv_heads=8, d=64, length=577, spread=0, page=16, causal=False, window=0),
        # single tokens of many sequences of uneven lengths, one of them empty, grouped heads
        dict(name="decode_batch", op="attend", qtype="q4_0", batch=32, nq=1, heads=32, kv_heads=8, d=128, length=16384, spread=15000, page=64, causal=False, window=0),
        # one token of one very long sequence: the work has to be split over the tokens
        dict(name="decode_long_q4_1", op="attend", qtype="q4_1", batch=1, nq=1, heads=16, kv_heads=2, d=128, length=524288, spread=0, page=64, causal=False, window=0),
        # a few tokens at once per sequence (checking a draft) in 8 bits, a sliding window that ends inside pages
        dict(name="verify_window_q8", op="attend", qtype="q8_0", batch=9, nq=5, heads=12, kv_heads=4, d=64, length=2001, spread=1990, page=48, causal=True, window=1000),
        # the memory attention of one frame: every token of a 64 x 64 map over a full memory bank
        dict(name="track_frame", op="attend", qtype="q4_0", batch=1, nq=4096, heads=1, kv_heads=1, d=256, length=28736, spread=0, page=64, causal=False, window=0),
        # a chunk of a long prompt over what is cached, causal, uneven lengths
        dict(name="prefill_chunk_q4_1", op="attend", qtype="q4_1", batch=4, nq=2048, heads=16, kv_heads=4, d=128, length=8191, spread=5000, page=64, causal=True, window=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = [work(c) for c in listed()]
    most = {k: max(w[k] for w in most) for k in ("bytes", "flops")}
    while True:
        op = rng.choice(["write", "read", "attend", "attend", "attend"])
        qtype = rng.choice(sorted(QTYPES))
        d = rng.choice([64, 128, 256])
        page = 16 * _log(rng, 1, 16)
        if op != "attend":
            n = _log(rng, 1, 65536)
            c = dict(op=op, qtype=qtype, n=n, heads=_log(rng, 1, 16), d=d, page=page, order=rng.choice(["pages", "any"]), dst=rng.choice(["f16", "f32"]))
            c["slots"] = -(-max(n, _log(rng, 16, 65536)) // page) * page
            if op == "write":
                c["src"] = rng.choice(["f16", "f32"])
            else:
                c["skip"] = rng.choice([0, 5])
        else:
            kv = _log(rng, 1, 16)
            nq = rng.choice([1, _log(rng, 1, 16), _log(rng, 16, 4096)])
            length = _log(rng, 1, 524288)
            c = dict(op=op, qtype=qtype, batch=_log(rng, 1, 32), nq=nq, heads=kv * rng.choice([1, 2, 3, 4, 8]), kv_heads=kv,
                     d=d, length=length, spread=rng.choice([0, int(length * rng.random())]), page=page,
                     causal=rng.random() < 0.6, window=0)
            if c["causal"] and rng.random() < 0.3:
                c["window"] = _log(rng, 16, 4096)
            # what the plain form holds: one score per query head and token, and the unpacked rows, in 32 bits
            if c["batch"] * c["heads"] * nq * length > 1.2e9 or c["batch"] * kv * length * d > 1.2e9:
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


def work(case):
    d, row = case["d"], _row_bytes(case)
    size = {"f16": 2, "f32": 4}
    if case["op"] == "attend":
        nq, heads = case["nq"], case["heads"]
        pairs = seen = 0
        for n in _lengths(case):
            first, last = _range(case, n, 0)[0], _range(case, n, nq - 1)[1]
            seen += max(0, last - first)
            if case["causal"] and nq * n:
                pairs += sum(max(0, hi - lo) for lo, hi in (_range(case, n, i) for i in range(nq)))
            else:
                pairs += nq * n
        io = 2 * 2 * case["batch"] * nq * heads * d
        return {"bytes": 2 * seen * case["kv_heads"] * row + io, "flops": 4 * d * heads * pairs}
    n, rows = case["n"], 2 * case["n"] * case["heads"]
    moved = rows * row + rows * d * size[case["dst"]] + 8 * n
    if case["op"] == "write":
        moved += rows * row + rows * d * size[case["src"]]
    return {"bytes": moved, "flops": rows * d * (6 if case["op"] == "write" else 2)}


def _range(case, n, i):
    """Positions [lo, hi) that query i sees in a sequence of n tokens."""
    if not case["causal"]:
        return 0, n
    hi = n - case["nq"] + i + 1
    lo = max(0, hi - case["window"]) if case["window"] else 0
    return lo, max(hi, 0)


# ------------------------------------------------------------------------------------------------ inputs
def _inputs(case, seed):
    """The tensors of a case, from the seed alone. Keys have channels of uneven size and offset, as projected keys do."""
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    d = case["d"]
    kv = case["kv_heads"] if case["op"] == "attend" else case["heads"]

    def rand(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    def kv_rows(n, dtype):
        k = rand(n, kv, d).mul_(torch.exp(0.4 * rand(1, kv, d))).add_(0.7 * rand(1, kv, d))
        v = rand(n, kv, d).mul_(torch.exp(0.4 * rand(1, kv, 1)))
        return k.to(dtype), v.to(dtype)

    if case["op"] == "attend":
        lengths = _lengths(case)
        per = -(-case["length"] // case["page"])
        total = case["batch"] * per
        pages = torch.randperm(total, device=dev, generator=g).to(torch.int32).view(case["batch"], per)
        k, v = kv_rows(total * case["page"], torch.float16)
        q = (0.8 * rand(case["batch"], case["nq"], case["heads"], d)).half()
        return dict(k=k, v=v, q=q, pages=pages, lengths=torch.tensor(lengths, dtype=torch.int32, device=dev))
    if case["order"] == "pages":  # consecutive tokens over the pages that a sequence was given, the first from its middle
        pages = torch.randperm(case["slots"] // case["page"], device=dev, generator=g)
        slots = (pages[:, None] * case["page"] + torch.arange(case["page"], device=dev)).flatten()
        first = min(case["page"] // 2 - 1, case["slots"] - case["n"])
        slots = slots[first:first + case["n"]].contiguous()
    else:
        slots = torch.randperm(case["slots"], device=dev, generator=g)[:case["n"]]
    if case["op"] == "write":
        k, v = kv_rows(case["n"], DTYPES[case["src"]])
    else:
        k, v = kv_rows(case["slots"], torch.float16)
        if case["skip"]:
            slots[case["skip"] - 1::case["skip"]] = -1
    return dict(k=k, v=v, slots=slots)


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
    kv = x["k"].shape[1]
    d, page = case["d"], case["page"]
    n_slots = case["slots"] if case["op"] != "attend" else x["k"].shape[0]
    state = {"case": case, **{n: x[n] for n in ("q", "pages", "lengths", "slots") if n in x}}
    if case["op"] == "write":
        state.update(k=x["k"], v=x["v"])
    else:
        every = torch.arange(n_slots, device="cuda")
    if case["op"] == "attend":
        state["scale"] = d ** -0.5
        state["out"] = torch.empty_like(x["q"])
    else:
        state["k_out"], state["v_out"] = (torch.empty(case["n"], kv, d, dtype=DTYPES[case["dst"]], device="cuda") for _ in "kv")
    # the cache that a program holds: the framework's own, or plain tensors of codes, scales and minima
    if own:
        s3b, eng = _framework()
        state["engine"] = eng
        state["cache"] = s3b.KVCache(QTYPES[case["qtype"]], n_slots // page, page, kv, d)
        if case["op"] != "write":
            eng.cache_write(state["cache"], x["k"], x["v"], every)
    else:
        state["cache"] = [_empty(case["qtype"], n_slots, kv, d) for _ in "kv"]
        if case["op"] != "write":
            for part, rows in zip(state["cache"], (x["k"], x["v"])):
                _store(case["qtype"], part, rows, every)
    torch.cuda.synchronize()
    return state


# ------------------------------------------------------------------------------------------------ plain form
def _empty(qtype, n, heads, d):
    code = torch.int8 if qtype == "q8_0" else torch.uint8
    scales = [torch.zeros(n, heads, d // 32, 1, dtype=torch.float16, device="cuda") for _ in range(2 if qtype == "q4_1" else 1)]
    return [torch.zeros(n, heads, d // 32, 32, dtype=code, device="cuda"), *scales]


def _over(x, by):
    """x / by rounded once: the division by a number multiplies by its rounded reciprocal on the GPU."""
    return x / torch.full_like(x, by)


def _quantise(qtype, rows):
    """Codes, scale (and minimum) of rows [n, heads, d], in the formats' own float32 steps."""
    x = torch.nan_to_num(rows.float(), nan=0.0, posinf=LIMIT, neginf=-LIMIT).clamp(-LIMIT, LIMIT)
    x = x.unflatten(-1, (-1, 32))
    if qtype == "q4_1":
        low = x.amin(-1, keepdim=True)
        scale = _over(x.amax(-1, keepdim=True) - low, 15.0)
        inv = torch.where(scale != 0, 1.0 / scale, 0.0)
        return ((x - low) * inv + 0.5).clamp(0, 15).to(torch.uint8), scale.half(), low.half()
    size = x.abs()
    peak = size.amax(-1, keepdim=True)
    if qtype == "q8_0":
        scale = _over(peak, 127.0)
        inv = torch.where(scale != 0, 1.0 / scale, 0.0)
        y = x * inv
        whole = y.trunc()
        return (whole + torch.where((y - whole).abs() >= 0.5, y.sign(), 0.0)).to(torch.int8), scale.half()
    # q4_0 scales by the value of largest magnitude with its sign, the first of equals
    place = torch.arange(32, device=x.device).expand_as(x)
    first = torch.where(size == peak, place, 32).amin(-1, keepdim=True)
    scale = torch.where(place == first, x, 0.0).sum(-1, keepdim=True) / -8.0
    inv = torch.where(scale != 0, 1.0 / scale, 0.0)
    return (x * inv + 8.5).clamp(0, 15).to(torch.uint8), scale.half()


def _store(qtype, part, rows, slots):
    for held, new in zip(part, _quantise(qtype, rows)):
        held[slots] = new


def _load(qtype, part, slots):
    """Rows of the given slots as float32 [..., heads, d]; a negative slot reads zeros."""
    codes, scale, *low = (t[slots.clamp(min=0)].float() for t in part)
    x = (codes - 8.0) * scale if qtype == "q4_0" else codes * scale
    if low:
        x = x + low[0]
    x = x.flatten(-2)
    return torch.where((slots >= 0)[..., None, None], x, 0.0)


def _attend(state):
    case, q = state["case"], state["q"].float()
    page, kv, d, nq = case["page"], case["kv_heads"], case["d"], case["nq"]
    at = torch.arange(case["length"], device="cuda")
    slots = state["pages"].long()[:, at // page] * page + at % page
    k, v = (_load(case["qtype"], part, slots) for part in state["cache"])         # [batch, tokens, kv heads, d]
    q = q.view(case["batch"], nq, kv, -1, d).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [batch, kv heads, group * nq, d]
    s = torch.matmul(q, k.permute(0, 2, 3, 1)) * state["scale"]
    length = state["lengths"].long()[:, None, None]
    seen = (at < length).expand(-1, nq, -1)
    if case["causal"]:
        end = length - nq + torch.arange(1, nq + 1, device="cuda")[None, :, None]
        seen = seen & (at < end)
        if case["window"]:
            seen = seen & (at >= end - case["window"])
    seen = seen[:, None, None]                                                      # [batch, 1, 1, nq, tokens]
    s = torch.where(seen, s.unflatten(2, (-1, nq)), -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), v.permute(0, 2, 1, 3)).unflatten(2, (-1, nq))
    o = o / torch.where(total == 0, 1.0, total)
    return o.permute(0, 3, 1, 2, 4).flatten(2, 3).half()


def run(state):
    case = state["case"]
    if own:
        eng, cache = state["engine"], state["cache"]
        if case["op"] == "attend":
            eng.cache_attention(cache, state["q"], state["out"], state["pages"], state["lengths"], state["scale"],
                                causal=case["causal"], window=case["window"])
            return state["out"]
        if case["op"] == "write":
            eng.cache_write(cache, state["k"], state["v"], state["slots"])
        eng.cache_read(cache, state["slots"], state["k_out"], state["v_out"])
        return state["k_out"], state["v_out"]
    if case["op"] == "attend":
        return _attend(state)
    if case["op"] == "write":
        _store(case["qtype"], state["cache"][0], state["k"], state["slots"])
        _store(case["qtype"], state["cache"][1], state["v"], state["slots"])
    return tuple(_load(case["qtype"], part, state["slots"]).to(DTYPES[case["dst"]]) for part in state["cache"])


# ------------------------------------------------------------------------------------------------ 64 bits
def _held(qtype, rows):
    """The values that rows [..., d] stand for once quantised, in 64 bits. The formats define their codes by float32
    steps, so each of those steps is taken exactly in 64 bits and then rounded to 32."""
    def f32(t):
        return t.float().double()
    x = rows.double().reshape(-1, 32)
    if qtype == "q4_1":
        low, high = x.min(1, keepdim=True).values, x.max(1, keepdim=True).values
        step = f32(f32(high - low) / 15)
    elif qtype == "q8_0":
        step = f32(x.abs().max(1, keepdim=True).values / 127)
    else:
        order = x.abs().sort(dim=1, descending=True, stable=True).indices[:, :1]
        step = x.gather(1, order) / -8
    inv = torch.zeros_like(step)
    inv[step != 0] = f32(1 / step[step != 0])
    kept = step.half().double()
    if qtype == "q4_1":
        code = f32(f32(f32(x - low) * inv) + 0.5).floor().clamp(max=15)
        y = code * kept + low.half().double()
    elif qtype == "q8_0":
        y = f32(x * inv)
        y = torch.copysign((y.abs() + 0.5).floor(), y) * kept
    else:
        y = (f32(f32(x * inv) + 8.5).floor().clamp(max=15) - 8) * kept
    return y.view(rows.shape)


def exact(case, seed):
    x = _inputs(case, seed)
    qtype = case["qtype"]
    if case["op"] == "write":
        return _held(qtype, x["k"]), _held(qtype, x["v"])
    if case["op"] == "read":
        out = []
        for rows in (x["k"], x["v"]):
            y = torch.zeros(case["n"], case["heads"], case["d"], dtype=torch.float64, device="cuda")
            use = x["slots"] >= 0
            y[use] = _held(qtype, rows[x["slots"][use]])
            out.append(y)
        return tuple(out)
    nq, page, group = case["nq"], case["page"], case["heads"] // case["kv_heads"]
    out = torch.zeros(case["batch"], nq, case["heads"], case["d"], dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(case)):
        if not n:
            continue
        slots = (x["pages"][b].long()[:, None] * page + torch.arange(page, device="cuda")).flatten()[:n]
        spans = torch.tensor([_range(case, n, i) for i in range(nq)], device="cuda")
        at = torch.arange(n, device="cuda")
        for h in range(case["kv_heads"]):
            k, v = _held(qtype, x["k"][slots, h]), _held(qtype, x["v"][slots, h])
            for first in range(0, nq, 1024):
                rows = slice(first, min(nq, first + 1024))
                hide = (at < spans[rows, :1]) | (at >= spans[rows, 1:])
                for m in range(h * group, (h + 1) * group):
                    s = (x["q"][b, rows, m].double() @ k.T) * case["d"] ** -0.5
                    p = s.masked_fill(hide, -math.inf).softmax(-1)
                    out[b, rows, m] = p.nan_to_num(0.0) @ v
    return out
