"""Serving over a paged key/value store: sequences of different lengths share one
pool of pages, their prompts enter it in chunks, and each then decodes token by
token, with full attention and under a sliding window with first tokens that stay
visible.  A second store of 16-bit pages over the values that the codes stand for
checks every step.

    python kivi-cache-rs_b200/examples/paged_serving.py [16|8|4]
"""
import math
import os
import sys

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

import torch  # noqa: E402

import kivi_cache as K  # noqa: E402


class Pool:
    """A store, its free pages and its sequences' block table."""

    def __init__(self, config, sequences, width):
        data, params = config.sizes()
        self.config = config
        self.memory = [torch.zeros(data, dtype=torch.uint8, device="cuda") for _ in range(2)]
        self.params = [torch.zeros(params, device="cuda") if params else None for _ in range(2)]
        self.pages = K.KvPages(config, *self.memory, *self.params)
        self.free = list(range(config.num_pages))
        self.table = torch.full((sequences, width), -1, dtype=torch.int32)
        self.lengths = [0] * sequences

    def batch(self, new):
        """Gives each sequence the pages that `new` more tokens need and returns the
        step's batch."""
        page = self.config.page_size
        for i, n in enumerate(new):
            for j in range(-(-self.lengths[i] // page), -(-(self.lengths[i] + n) // page)):
                self.table[i, j] = self.free.pop()
            self.lengths[i] += n
        cu = torch.tensor([0] + new, dtype=torch.int32).cumsum(0).to(torch.int32)
        return K.PagesBatch(self.table.cuda(), cu.cuda(), torch.tensor(self.lengths, dtype=torch.int32).cuda(), sum(new), max(new))


def serve(bits=8, sequences=4, prompt=1000, steps=8, chunk=64, kv_heads=2, q_heads=8, dim=128, page_size=32, window=256,
          sinks=4):
    """Largest difference of any output from the check's."""
    torch.manual_seed(0)
    width = -(-(prompt + steps) // page_size)
    sizes = dict(num_pages=sequences * width, page_size=page_size, num_kv_heads=kv_heads, head_dim=dim)
    pool = Pool(K.PagesConfig(bits=bits, **sizes), sequences, width)
    check = Pool(K.PagesConfig(bits=16, **sizes), sequences, width)
    scale, worst = 1.0 / math.sqrt(dim), 0.0
    left = [prompt - 37 * i for i in range(sequences)]  # prompts of different lengths
    done = [0] * sequences
    while min(done) < steps:
        # a sequence with prompt left takes a chunk of it, the others decode one token
        new = [min(chunk, n) if n else 1 for n in left]
        done = [d + (n == 0) for d, n in zip(done, left)]
        left = [n - min(chunk, n) for n in left]
        if max(done) > steps:
            break
        total = sum(new)
        k, v = (torch.randn(total, kv_heads, dim, device="cuda").bfloat16() for _ in range(2))
        q = torch.randn(total, q_heads, dim, device="cuda").bfloat16()
        batch, other = pool.batch(new), check.batch(new)
        pool.pages.write_dev(batch, k, v)
        pool.pages.read_dev(batch, k, v)  # what the later steps will see
        check.pages.write_dev(other, k, v)
        for w in (0, window):
            out, want = torch.empty_like(q), torch.empty_like(q)
            pool.pages.attention_dev(batch, q, q_heads, scale, out, window=w, sinks=sinks)
            check.pages.attention_dev(other, q, q_heads, scale, want, window=w, sinks=sinks)
            worst = max(worst, float((out.float() - want.float()).abs().max()))
    pool.pages.status()
    check.pages.status()
    return worst


if __name__ == "__main__":
    width = int(sys.argv[1]) if len(sys.argv) > 1 else 8
    print(f"{width}-bit pages: largest difference from 16-bit pages of the same values {serve(width):.4f}")
