"""A memory of the last frames of a stream as a quantised key / value cache.

Every frame leaves a feat x feat map of 64-channel features and a few pointer tokens. Their keys and values (one head of 256)
are projected once, with random weights here, quantised into the pages of a ring of the last `slots` frames, and every new
frame attends over what the ring holds: the page table lists the pages of the frames to look at, so a frame is dropped or
reused by changing the table, and a page can be read back or copied out as it is. This holds for keys that stay as they
are once written. The engine's own tracking step adds an encoding of a frame's age to its keys, which would have to be
written anew each frame, and keeps the 64 channels instead.

  python examples/stream_memory.py [--feat 64] [--frames 12] [--slots 7] [--type q4_0]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
from __graft_entry__ import _pkg  # noqa: E402

TYPES = {"q4_0": 2, "q4_1": 3, "q8_0": 8}


class StreamMemory:
    """Memory of `slots` frames of feat * feat map tokens and `pointers` pointer tokens each."""

    D = 256

    def __init__(self, s3b, engine, feat, slots=7, pointers=4, qtype=2, page=64, seed=0):
        self.engine, self.tokens, self.page = engine, feat * feat + pointers, page
        self.pages_of_frame = -(-self.tokens // page)
        self.cache = s3b.KVCache(qtype, slots * self.pages_of_frame, page, 1, self.D)
        self.slots, self.frames = slots, []  # ring slots in the order in which they were written
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.w_k, self.w_v = ((torch.randn(self.D, 64, device="cuda", generator=g) / 8).half() for _ in "kv")
        self.k, self.v = (torch.empty(self.tokens, 1, self.D, device="cuda", dtype=torch.float16) for _ in "kv")

    def slot_rows(self, ring_slot):
        """Cache slots of a ring slot's tokens."""
        first = ring_slot * self.pages_of_frame * self.page
        return torch.arange(first, first + self.tokens, device="cuda")

    def write(self, features):
        """Projects the memory features f16 [tokens, 64] of a frame and quantises them over the oldest frame."""
        ring_slot = len(self.frames) if len(self.frames) < self.slots else self.frames.pop(0)
        self.engine.gemm(features, self.w_k, self.k.view(self.tokens, self.D))
        self.engine.gemm(features, self.w_v, self.v.view(self.tokens, self.D))
        self.engine.cache_write(self.cache, self.k, self.v, self.slot_rows(ring_slot))
        self.frames.append(ring_slot)

    def attend(self, q):
        """Attention of q f16 [n, 256] over each frame of the ring: a sequence a frame, joined by their sums (a frame's tokens
        end inside its last page, so the frames are not one run of full pages)."""
        n, f = q.shape[0], len(self.frames)
        pages = (torch.tensor(self.frames, dtype=torch.int32, device="cuda")[:, None] * self.pages_of_frame +
                 torch.arange(self.pages_of_frame, dtype=torch.int32, device="cuda")).contiguous()
        lengths = torch.full((f,), self.tokens, dtype=torch.int32, device="cuda")
        out = torch.empty(f, n, 1, self.D, device="cuda")
        lse = torch.empty(f, n, 1, device="cuda")
        self.engine.cache_attention(self.cache, q.view(1, n, 1, self.D).expand(f, n, 1, self.D), out, pages, lengths,
                                    self.D ** -0.5, lse=lse)
        return (out * torch.softmax(lse, 0)[..., None]).sum(0).view(n, self.D)

    def read(self):
        """Keys and values of all frames as the cache holds them, oldest first."""
        rows = torch.cat([self.slot_rows(s) for s in self.frames])
        k, v = (torch.empty(len(rows), 1, self.D, device="cuda") for _ in "kv")
        self.engine.cache_read(self.cache, rows, k, v)
        return k.view(-1, self.D), v.view(-1, self.D)


def run(feat=64, frames=12, slots=7, qtype=2, seed=0):
    """Streams random frames; returns the attention of the last one over the memory, the same in 64 bits on the values that
    the cache holds and on the unquantised ones, and the bytes of the cache and of f16 keys and values for its tokens."""
    s3b = _pkg()
    engine = s3b.Engine(0)
    engine.set_stream(torch.cuda.current_stream().cuda_stream)
    memory = StreamMemory(s3b, engine, feat, slots, qtype=qtype, seed=seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    kept = []
    for _ in range(frames):
        features = torch.randn(memory.tokens, 64, device="cuda", generator=g).half()
        memory.write(features)
        kept = (kept + [features])[-slots:]
        q = torch.randn(feat * feat, memory.D, device="cuda", generator=g).half()
        out = memory.attend(q)
    engine.sync()

    def exact(k, v):
        s = q.double() @ k.double().T * memory.D ** -0.5
        return s.softmax(-1) @ v.double()
    held = exact(*memory.read())
    engine.sync()
    features = torch.cat(kept).double()
    full = exact(features @ memory.w_k.double().T, features @ memory.w_v.double().T)
    sizes = memory.cache.data.numel(), 2 * slots * memory.tokens * memory.D * 2
    engine.close()
    return out, held, full, sizes


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--feat", type=int, default=64)
    ap.add_argument("--frames", type=int, default=12)
    ap.add_argument("--slots", type=int, default=7)
    ap.add_argument("--type", choices=sorted(TYPES), default="q4_0")
    a = ap.parse_args()
    out, held, full, (cache, plain) = run(a.feat, a.frames, a.slots, TYPES[a.type])

    def off(x, y):
        return ((x.double() - y).norm() / y.norm()).item()
    print(f"{a.type}: {cache / 2 ** 20:.1f} MiB for {plain / 2 ** 20:.1f} MiB of f16 keys and values; attention off by "
          f"{off(out, held):.1e} from 64 bits on the values held, by {off(out, full):.1e} from the unquantised ones")


if __name__ == "__main__":
    main()
