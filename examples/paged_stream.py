"""A stack of attention layers served from the paged 8-bit K/V cache: prompts of different lengths in one step, then
single tokens in a captured step, a request that ends and one that takes its place.

    python examples/paged_stream.py [--layers 4 --requests 8 --steps 32]

The layers are random projections with grouped heads; what counts is the order of the calls.  At the end the last step's
outputs are held against the same layers over exact keys and values, and the step's time and the cache's size are printed.
"""

from __future__ import annotations

import argparse
import pathlib
import sys

import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1] / "minicpm-o-4.5-single-gpu-engine_b200"))

from b200t2w.paged import B200PagedCache  # noqa: E402

PAGE, Q_HEADS, KV_HEADS, HEAD_DIM = 16, 16, 4, 64
WIDTH = Q_HEADS * HEAD_DIM
GROUP = Q_HEADS // KV_HEADS


class Stack:
    """Layers of x + attend(q, k, v) out; ``kept`` holds every layer's exact keys and values for the comparison."""

    def __init__(self, layers: int):
        gen = torch.Generator(device="cuda").manual_seed(0)
        qkv = (Q_HEADS + 2 * KV_HEADS) * HEAD_DIM

        def weight(n, m):
            return (torch.randn(n, m, device="cuda", generator=gen) * m ** -0.5).bfloat16()

        self.qkv = [weight(qkv, WIDTH) for _ in range(layers)]
        self.out = [weight(WIDTH, WIDTH) for _ in range(layers)]
        self.kept = None

    def __call__(self, x: torch.Tensor, cache: B200PagedCache, plan) -> torch.Tensor:
        for i, (w, o) in enumerate(zip(self.qkv, self.out)):
            q, k, v = self.heads(x, w)
            cache.append(i, k, v, plan)
            x = x + cache.attend(i, q, plan).view(-1, WIDTH) @ o.T
            if self.kept is not None:
                self.kept.append((k.clone(), v.clone()))
        return x

    @staticmethod
    def heads(x: torch.Tensor, w: torch.Tensor):
        """Queries, keys and values as views of the fused projection's rows."""
        rows = (x.float() * x.float().pow(2).mean(-1, keepdim=True).add(1e-6).rsqrt()).to(x.dtype) @ w.T
        return rows.view(-1, Q_HEADS + 2 * KV_HEADS, HEAD_DIM).split([Q_HEADS, KV_HEADS, KV_HEADS], dim=1)

    def exact(self, x: torch.Tensor, history) -> torch.Tensor:
        """One new row over a layer's keys and values ``history[layer]``, in fp32."""
        for i, (w, o) in enumerate(zip(self.qkv, self.out)):
            q, k, v = (t.float() for t in self.heads(x, w))
            k, v = (torch.cat([h.float(), t]).repeat_interleave(GROUP, 1) for h, t in zip(history[i], (k, v)))
            weight = torch.softmax(torch.einsum("rhd,nhd->hrn", q, k) * HEAD_DIM ** -0.5, -1)
            x = x + torch.einsum("hrn,nhd->rhd", weight, v).reshape(1, WIDTH).to(x.dtype) @ o.T
        return x


def run(layers: int = 4, requests: int = 8, steps: int = 32, say=print) -> float:
    """Serve, compare, and return the largest difference of the last step's outputs in units of their spread."""
    gen = torch.Generator(device="cuda").manual_seed(1)

    def rows(n):
        return torch.randn(n, WIDTH, device="cuda", generator=gen).bfloat16()

    def i32(x):
        return torch.tensor(x, device="cuda", dtype=torch.int32)

    prompts = [40 + 37 * r for r in range(requests)]
    longest = max(prompts) + steps + 4
    blocks = -(-longest // PAGE)
    cache = B200PagedCache(layers, requests * blocks, PAGE, KV_HEADS, HEAD_DIM, requests, longest, q_heads=Q_HEADS)
    stack = Stack(layers)

    # The prompts, all in one step: one plan for all layers.
    plan = cache.plan(i32(prompts), rows=sum(prompts), max_fresh=max(prompts))
    stack(rows(sum(prompts)), cache, plan)
    plan.check()  # (waits for the GPU; a server would look at it now and then)

    # Single tokens: the step is captured once, its plan's kernels with it, and replayed for every token.
    ones, x = i32([1] * requests), rows(requests)

    def step():
        p = cache.plan(ones, rows=requests, max_fresh=1)
        out = stack(x, cache, p)
        x.copy_(out / out.float().std().clamp_min(1.0))  # stands for the sampled tokens' embeddings
        return p

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # (makes the libraries' handles and workspaces; it is a token like any other)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = step()
    graph.replay()
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    for _ in range(steps):
        graph.replay()
    end.record()
    plan.check()
    say(f"{requests} requests, {layers} layers: {begin.elapsed_time(end) / steps * 1e3:.0f} us a step of {requests} tokens; "
        f"{cache.bytes_per_token()} bytes a token (bf16: {2 * cache.bytes_per_token()})")

    # Request 0 ends; its pages go back and another prompt takes its place while the others bring a token each.
    cache.release(i32([1] + [0] * (requests - 1)))
    cache.check()
    fresh = [65] + [1] * (requests - 1)
    stack.kept = []
    stack(rows(sum(fresh)), cache, cache.plan(i32(fresh), rows=sum(fresh), max_fresh=65))
    history, stack.kept = [(k[:65], v[:65]) for k, v in stack.kept], None  # the new request's, exact

    # Its next token, over the cache and over the exact keys and values.
    x = rows(requests)
    plan = cache.plan(ones, rows=requests, max_fresh=1)
    got, want = stack(x, cache, plan)[:1].float(), stack.exact(x[:1], history).float()
    plan.check()
    worst = ((got - want).abs().max() / want.std()).item()
    say(f"the new request's next token: within {worst:.3f} standard deviations of the layers over exact keys and values")
    return worst


if __name__ == "__main__":
    a = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    a.add_argument("--layers", type=int, default=4)
    a.add_argument("--requests", type=int, default=8)
    a.add_argument("--steps", type=int, default=32)
    run(**vars(a.parse_args()))
