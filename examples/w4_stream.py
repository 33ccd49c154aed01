"""A stack of decoder layers with 4-bit weights, rotary positions and the paged 8-bit K/V cache: prompts in one step, then single
tokens in a captured step.

    python examples/w4_stream.py [--layers 2 --requests 8 --steps 32]

The layers' weights are random; what counts is the order of the calls.  At the end the last step's outputs are held against the
same layers with the unrounded 16-bit products of torch over the same cache, and the step's time and the weights' size printed.
"""

from __future__ import annotations

import argparse
import pathlib
import sys

import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1] / "minicpm-o-4.5-single-gpu-engine_b200"))

from b200t2w import w4  # noqa: E402
from b200t2w.paged import B200PagedCache  # noqa: E402
from b200t2w.rotary import Rotary  # noqa: E402

PAGE, Q_HEADS, KV_HEADS, HEAD_DIM = 16, 16, 4, 64
WIDTH, HIDDEN = Q_HEADS * HEAD_DIM, 2816
HEADS = Q_HEADS + 2 * KV_HEADS


def norm(x: torch.Tensor) -> torch.Tensor:
    return (x.float() * x.float().pow(2).mean(-1, keepdim=True).add(1e-6).rsqrt()).to(x.dtype)


class Layer:
    """x + out(attention(rotary(qkv(norm x)))), then the gated feed-forward, every product with 4-bit weights."""

    def __init__(self, gen: torch.Generator):
        def quantized(n, k):
            return w4.quantize((torch.randn(n, k, device="cuda", generator=gen) * k ** -0.5).bfloat16(), 64, zeros=True)

        parts = [quantized(HEADS * HEAD_DIM, WIDTH), quantized(WIDTH, WIDTH), quantized(HIDDEN, WIDTH), quantized(HIDDEN, WIDTH),
                 quantized(WIDTH, HIDDEN)]
        self.qkv, self.out, self.gate_up, self.down = (w4.pack(*parts[0]), w4.pack(*parts[1]),
                                                       w4.pack_gated(parts[2], parts[3]), w4.pack(*parts[4]))
        self.dense = [w4.pack(*q).unpack().bfloat16() for q in parts]  # for the comparison alone

    def __call__(self, i, x, positions, turn, cache, plan):
        rows = w4.linear(norm(x), self.qkv).view(-1, HEADS, HEAD_DIM)
        q, k, v = rows.split([Q_HEADS, KV_HEADS, KV_HEADS], dim=1)
        turn.apply_(q, k, positions)  # in place, in the fused rows
        cache.append(i, k, v, plan)
        x = w4.linear(cache.attend(i, q, plan).view(-1, WIDTH), self.out, residual=x)
        return w4.feed_forward(norm(x), self.gate_up, self.down, residual=x)

    def plain(self, i, x, positions, turn, cache, plan):
        """The same with torch's products over 16-bit weights (rows appended already)."""
        qkv, out, gate, up, down = self.dense
        q = (norm(x) @ qkv.T).view(-1, HEADS, HEAD_DIM)[:, :Q_HEADS].contiguous()
        q, _ = turn(q, None, positions)
        x = x + cache.attend(i, q, plan).view(-1, WIDTH) @ out.T
        h = norm(x)
        return x + (torch.nn.functional.silu((h @ gate.T).float()) * (h @ up.T).float()).to(x.dtype) @ down.T


def run(layers: int = 2, requests: int = 8, steps: int = 32, say=print) -> float:
    """Serve, compare, and return the largest difference of the last step's outputs in units of their spread."""
    gen = torch.Generator(device="cuda").manual_seed(1)

    def rows(n):
        return torch.randn(n, WIDTH, device="cuda", generator=gen).bfloat16()

    def i32(x):
        return torch.tensor(x, device="cuda", dtype=torch.int32)

    prompts = [30 + 17 * r for r in range(requests)]
    longest = max(prompts) + steps + 4
    cache = B200PagedCache(layers, requests * -(-longest // PAGE), PAGE, KV_HEADS, HEAD_DIM, requests, longest, q_heads=Q_HEADS)
    stack, turn = [Layer(gen) for _ in range(layers)], Rotary(HEAD_DIM, [HEAD_DIM // 2], base=500000.0)

    plan = cache.plan(i32(prompts), rows=sum(prompts), max_fresh=max(prompts))
    x, at = rows(sum(prompts)), i32([p for n in prompts for p in range(n)])
    for i, layer in enumerate(stack):
        x = layer(i, x, at, turn, cache, plan)
    plan.check()

    ones, x = i32([1] * requests), rows(requests)

    def step():
        p = cache.plan(ones, rows=requests, max_fresh=1)
        positions, y = cache.length - 1, x
        for i, layer in enumerate(stack):
            y = layer(i, y, positions, turn, cache, p)
        return p, y

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # (makes the libraries' handles and workspaces; it is a token like any other)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan, y = step()
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    for _ in range(steps):
        graph.replay()
    end.record()
    plan.check()
    size = sum(w.buffer.numel() for layer in stack for w in (layer.qkv, layer.out, layer.gate_up, layer.down))
    say(f"{requests} requests, {layers} layers: {begin.elapsed_time(end) / steps * 1e3:.0f} us a step of {requests} tokens; "
        f"weights {size >> 10} KB (bf16: {sum(d.numel() for layer in stack for d in layer.dense) >> 9} KB)")

    # The last step's rows once more, against 16-bit products over the cache as that step left it.
    want = x
    for i, layer in enumerate(stack):
        want = layer.plain(i, want, cache.length - 1, turn, cache, plan)
    for layer in stack:
        for w in (layer.qkv, layer.out, layer.gate_up, layer.down):
            w.check()
    worst = ((y.float() - want.float()).abs().max() / want.float().std()).item()
    say(f"the last step's outputs: within {worst:.3f} standard deviations of 16-bit products")
    return worst


if __name__ == "__main__":
    a = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    a.add_argument("--layers", type=int, default=2)
    a.add_argument("--requests", type=int, default=8)
    a.add_argument("--steps", type=int, default=32)
    run(**vars(a.parse_args()))
