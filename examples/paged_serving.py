"""A serving loop over the paged KV cache: requests of different lengths join and
leave one batch, prompts are prefilled in chunks beside the decode steps of the
others, and every step is two calls for the whole batch: write the new tokens'
keys and values, then attend.

    python examples/paged_serving.py [--pages same|int8|e4m3] [--steps N] [--budget N]

With a budget every request's cache is cut to that many tokens whenever it has grown
a quarter beyond: the attention weight that each key received is summed over the
steps (``kvcache_weights_paged``), and those with the least go
(``kvcache_evict_paged``), but for the first four and the most recent.

The "model" is one attention layer with random projections and a token drawn
from its output, enough to have real data flow through the cache.  At the end
each request's last token is checked against attention over its own keys and
values read back from the cache (``kvcache_read_paged`` +
``flash_attention_varlen_forward``).  Needs a B200 and the in-tree build.
"""
import argparse
import os
import sys

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(REPO, "flash-attention-sm75-register-fused_b200"))

import torch  # noqa: E402

import flash_attention_sm75 as fa  # noqa: E402

HQ, HKV, D, PAGE, HIDDEN, VOCAB = 16, 4, 128, 16, 512, 997
PAGES = {"same": torch.bfloat16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}


class PagedCache:
    """Pages for one layer and the free list that hands them to requests."""

    def __init__(self, num_pages, kind, device):
        shape = (num_pages, HKV, PAGE, D)
        self.k = torch.empty(shape, dtype=kind, device=device)
        self.v = torch.empty(shape, dtype=kind, device=device)
        eight = self.k.element_size() == 1
        self.scales = dict(k_scale=torch.empty(shape[:3], device=device),
                           v_scale=torch.empty(shape[:3], device=device)) if eight else {}
        self.free = list(range(num_pages - 1, -1, -1))

    def grow(self, pages, length):
        """Extend a request's page list to hold `length` tokens."""
        while len(pages) * PAGE < length:
            pages.append(self.free.pop())

    def release(self, pages):
        self.free.extend(pages)
        pages.clear()


class Request:
    def __init__(self, prompt, new_tokens):
        self.todo = list(prompt)  # tokens not yet in the cache
        self.left = new_tokens    # tokens still to be drawn
        self.length = 0           # tokens in the cache
        self.pages = []
        self.drawn = []
        self.sums = None          # attention weight of its keys, where a budget asks for it


class Layer:
    def __init__(self, device, dtype=torch.bfloat16):
        g = torch.Generator(device=device).manual_seed(0)

        def weight(*shape):
            return (torch.randn(*shape, generator=g, device=device) / shape[0] ** 0.5).to(dtype)

        self.embed = weight(VOCAB, HIDDEN) * VOCAB ** 0.5
        self.qkv = weight(HIDDEN, (HQ + 2 * HKV) * D)
        self.out = weight(HQ * D, VOCAB)

    def project(self, tokens):
        x = (self.embed[tokens] @ self.qkv).view(-1, HQ + 2 * HKV, D)
        # slices of one projection: the cache and the attention read them in place
        return x[:, :HQ], x[:, HQ:HQ + HKV], x[:, HQ + HKV:]


def add_weights(cache, batch, q, lse, table, cu, lens, new):
    """Adds what the step's tokens gave to the batch's keys to the requests' sums."""
    held = table.size(1) * PAGE
    sums = torch.zeros(len(batch), HKV, held, device=q.device)
    for i, r in enumerate(batch):
        if r.sums is not None:
            n = min(held, r.sums.size(1))
            sums[i, :, :n] = r.sums[:, :n]
    fa.kvcache_weights_paged(q, lse, cache.k, table, cu, lens, max(len(n) for n in new),
                             max(r.length for r in batch), sums, causal=True,
                             k_scale=cache.scales.get("k_scale"))
    for i, r in enumerate(batch):
        r.sums = sums[i]


def evict(cache, batch, budget):
    """Cuts the caches that have grown a quarter beyond the budget."""
    full = [r for r in batch if r.length > budget + budget // 4]
    if not full:
        return
    dev = cache.k.device
    width = max(len(r.pages) for r in full)
    table = torch.tensor([r.pages + [-1] * (width - len(r.pages)) for r in full], dtype=torch.int32).to(dev)
    sums = torch.zeros(len(full), HKV, width * PAGE, device=dev)
    for i, r in enumerate(full):
        n = min(width * PAGE, r.sums.size(1))
        sums[i, :, :n] = r.sums[:, :n]
    lens = fa.kvcache_evict_paged(cache.k, cache.v, sums, table, [r.length for r in full], budget,
                                  recent=budget // 4, first=4, **cache.scales).tolist()
    for i, r in enumerate(full):
        r.length, r.sums = lens[i], sums[i]
        keep = -(-r.length // PAGE)
        cache.free.extend(r.pages[keep:])
        del r.pages[keep:]


def step(layer, cache, batch, chunk, budget=0):
    """One step of a batch: up to `chunk` prompt tokens, or one drawn token, of
    every request.  Returns the tokens drawn."""
    dev = cache.k.device
    new = [r.todo[:chunk] for r in batch]
    for r, n in zip(batch, new):
        r.todo = r.todo[len(n):]
        r.length += len(n)
        cache.grow(r.pages, r.length)
    width = max(len(r.pages) for r in batch)
    table = torch.tensor([r.pages + [-1] * (width - len(r.pages)) for r in batch],
                         dtype=torch.int32).to(dev)
    lens = torch.tensor([r.length for r in batch], dtype=torch.int32).to(dev)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + len(n))
    cu_dev = torch.tensor(cu, dtype=torch.int32).to(dev)
    q, k, v = layer.project(torch.tensor([t for n in new for t in n]).to(dev))
    fa.kvcache_write_paged(k, v, cache.k, cache.v, table, cu_dev, lens, **cache.scales)
    o, lse = fa.flash_attention_forward_paged(q, cache.k, cache.v, table, cu_dev, lens,
                                              max(len(n) for n in new), max(r.length for r in batch),
                                              causal=True, return_lse=True, **cache.scales)
    if budget:
        add_weights(cache, batch, q, lse, table, cu_dev, lens, new)
    last = o[torch.tensor(cu[1:]).to(dev) - 1].reshape(len(batch), HQ * D)
    drawn = (last @ layer.out).argmax(-1).tolist()
    for r, t in zip(batch, drawn):
        if not r.todo and r.left > 0:  # the prompt is through: the drawn token is next
            r.left -= 1
            r.drawn.append(t)
            r.todo = [t]
    return q, o, table, lens, cu


def check(cache, batch, q, o, table, lens, cu):
    """The step's last tokens against attention over the keys read back."""
    n = [r.length for r in batch]
    cu_k = [0]
    for x in n:
        cu_k.append(cu_k[-1] + x)
    k, v = fa.kvcache_read_paged(cache.k, cache.v, table, cu_k, lens, cu_k[-1], dtype=q.dtype, **cache.scales)
    rows = torch.tensor(cu[1:], device=q.device) - 1
    ref = fa.flash_attention_varlen_forward(q[rows].contiguous(), k, v, list(range(len(batch) + 1)), cu_k, 1,
                                            max(n), causal=True)
    return (ref.float() - o[rows].float()).abs().max().item()


def serve(pages="int8", steps=40, chunk=96, device="cuda", verbose=True, budget=0):
    """Runs the loop; returns (tokens drawn per request, largest difference seen)."""
    cache = PagedCache(512, PAGES[pages], device)
    layer = Layer(device)
    g = torch.Generator().manual_seed(1)

    def request(n, new):
        return Request(torch.randint(VOCAB, (n,), generator=g).tolist(), new)

    waiting = [request(n, new) for n, new in ((300, 12), (7, 30), (1000, 8), (45, 20), (160, 4))]
    batch, done, worst = [], [], 0.0
    for i in range(steps):
        if waiting and len(batch) < 4:
            batch.append(waiting.pop(0))
        state = step(layer, cache, batch, chunk, budget)
        worst = max(worst, check(cache, batch, *state))
        if verbose:
            print(f"step {i:2d}: {len(batch)} requests, {state[4][-1]:3d} new tokens, "
                  f"{sum(r.length for r in batch):4d} cached")
        if budget:
            evict(cache, batch, budget)
        for r in [r for r in batch if not r.todo]:
            batch.remove(r)
            cache.release(r.pages)
            done.append(r)
        if not batch and not waiting:
            break
    if verbose:
        print(f"largest difference from attention over the keys read back: {worst:.2e}")
    return [r.drawn for r in done], worst


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--pages", choices=sorted(PAGES), default="int8")
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--budget", type=int, default=0)
    args = ap.parse_args()
    serve(args.pages, args.steps, budget=args.budget)
