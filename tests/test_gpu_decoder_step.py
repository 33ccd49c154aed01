"""GPU: a decoder layer's step made of the operators together: the fused projection with 4-bit weights, rotary positions in place in
its rows, the paged cache's append and attention, the output projection onto the residual stream and the gated feed-forward; each
part held against the plain statement on the very inputs that it got, and the captured step against the eager one."""

import importlib.util
import math
import pathlib

import pytest
import torch

import w4_ref as ref
from b200t2w import lib as L
from b200t2w import w4
from b200t2w.paged import B200PagedCache
from b200t2w.rotary import Rotary
from test_gpu_paged import attention as plain_attention

pytestmark = pytest.mark.gpu

HEADS, KV, HD, HIDDEN, PAGE = 8, 2, 64, 1088, 16
WIDTH, ALL = HEADS * HD, HEADS + 2 * KV


@pytest.fixture(scope="module", autouse=True)
def _dev():
    assert torch.cuda.is_available()
    assert L.load().t2w_device_ok(torch.cuda.current_device()) == 1


def cuda(w):
    return tuple(None if t is None else t.cuda() for t in w)


def held(out, want):
    y, lim = want
    d = (out.double().cpu() - y).abs()
    assert out.shape == y.shape and bool((d <= lim).all()), float((d / lim).max())


class Step:
    def __init__(self, seed):
        gen = torch.Generator().manual_seed(seed)
        self.qkv = ref.weights(ALL * HD, WIDTH, 64, True, torch.bfloat16, gen)
        self.out = ref.weights(WIDTH, WIDTH, 128, False, torch.bfloat16, gen)
        self.gate, self.up = (ref.weights(HIDDEN, WIDTH, 32, True, torch.bfloat16, gen) for _ in range(2))
        self.down = ref.weights(WIDTH, HIDDEN, 64, True, torch.bfloat16, gen)
        self.p_qkv, self.p_out, self.p_down = (w4.pack(*cuda(w)) for w in (self.qkv, self.out, self.down))
        self.p_gate_up = w4.pack_gated(cuda(self.gate), cuda(self.up))
        self.turn = Rotary(HD, [12, 10, 10], base=10000.0)

    def __call__(self, x, positions, cache, plan):
        rows = w4.linear(x, self.p_qkv)
        before = rows.clone()
        q, k, v = rows.view(-1, ALL, HD).split([HEADS, KV, KV], dim=1)
        self.turn.apply_(q, k, positions)
        cache.append(0, k, v, plan)
        a = cache.attend(0, q, plan).view(-1, WIDTH)
        y = w4.linear(a, self.p_out, residual=x)
        h = w4.gated(y, self.p_gate_up)
        return before, rows, a, y, h, w4.linear(h, self.p_down, residual=y)


def cache_of(requests, tokens):
    return B200PagedCache(1, requests * -(-tokens // PAGE), PAGE, KV, HD, requests, tokens, q_heads=HEADS)


@pytest.mark.parametrize("fresh", [[1], [1, 1, 1, 1, 1], [9, 1, 30, 0, 7], [100, 60]])
def test_parts(fresh):
    step, gen = Step(len(fresh)), torch.Generator().manual_seed(sum(fresh))
    rows, cache = sum(fresh), cache_of(len(fresh), 300)
    f = torch.tensor(fresh, dtype=torch.int32, device="cuda")
    axis = torch.tensor([0] * 12 + [1] * 10 + [2] * 10)
    freq = torch.tensor([10000.0 ** (-2 * i / HD) for i in range(32)], dtype=torch.float64)
    for turn in range(2):  # prompts, and the same again behind them
        x = torch.randn(rows, WIDTH, generator=gen).bfloat16()
        positions = torch.randint(0, 4000, (3, rows), generator=gen)
        plan = cache.plan(f, rows=rows, max_fresh=max(fresh))
        before, after, a, y, h, z = step(x.cuda(), positions.cuda(), cache, plan)
        plan.check()
        held(before, ref.linear(x, step.qkv))
        turned = ref.turned(before.cpu().view(rows, ALL, HD)[:, :HEADS + KV], positions, axis, freq, HD, False, False)
        size = before.cpu().double().view(rows, ALL, 2, HD // 2)[:, :HEADS + KV].abs().sum(2, keepdim=True)
        error = 2.0 ** -21 * size.expand(-1, -1, 2, -1).reshape(turned.shape)
        held(after.view(rows, ALL, HD)[:, :HEADS + KV], (turned, ref.rounded(turned, error, torch.bfloat16)))
        assert torch.equal(after.view(rows, ALL, HD)[:, HEADS + KV:], before.view(rows, ALL, HD)[:, HEADS + KV:])
        assert bool(torch.isfinite(a).all())
        held(y, ref.linear(a.cpu(), step.out, None, x))
        held(h, ref.gated(y.cpu(), step.gate, step.up, "silu"))
        held(z, ref.linear(h.cpu(), step.down, None, y.cpu()))
    for p in (step.p_qkv, step.p_out, step.p_gate_up, step.p_down):
        p.check()


@pytest.mark.parametrize("fresh", [[1], [9, 1, 30, 0, 7], [100, 60]])
def test_attention_of_the_step(fresh):
    """The step's attention against the plain one over what its cache holds, and what it holds against the turned keys and the
    values of the fused rows.

    The attention's bound is that of ``test_gpu_paged``.  A cached value is rounded to e4m3 once, and once more where a later row
    raises its page's scale: twice half a step, 2^-4 of the value or 2^-10 of the scale, the second of what the first left."""
    step, gen = Step(len(fresh) + 20), torch.Generator().manual_seed(sum(fresh) + 1)
    rows, cache = sum(fresh), cache_of(len(fresh), 300)
    f = torch.tensor(fresh, dtype=torch.int32, device="cuda")
    told = [[[] for _ in fresh] for _ in range(2)]  # keys and values of each request
    for _ in range(2):
        x = torch.randn(rows, WIDTH, generator=gen).bfloat16()
        positions = torch.randint(0, 4000, (3, rows), generator=gen)
        plan = cache.plan(f, rows=rows, max_fresh=max(fresh))
        _, after, a, *_ = step(x.cuda(), positions.cuda(), cache, plan)
        plan.check()
        after = after.double().cpu().view(rows, ALL, HD)
        out = a.double().cpu().view(rows, HEADS, HD)
        table, start = cache.table.cpu(), 0
        codes = [t[0].float().double().cpu() * s[0].double().cpu()[..., None, None] for t, s in
                 ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]
        scale = [s[0].double().cpu() for s in (cache.k_scale, cache.v_scale)]
        for r, n in enumerate(fresh):
            part = after[start:start + n]
            held_rows = []
            for w in range(2):
                told[w][r].append(part[:, HEADS + w * KV:HEADS + (w + 1) * KV])
                want = torch.cat(told[w][r])
                pages = table[r, :-(-want.shape[0] // PAGE)].long()
                got = codes[w][pages].transpose(1, 2).reshape(-1, KV, HD)[:want.shape[0]]
                each = scale[w][pages].repeat_interleave(PAGE, 0)[:want.shape[0], :, None]
                once = 2.0 ** -4 * want.abs() + 2.0 ** -10 * each
                assert bool(((got - want).abs() <= once + 2.0 ** -4 * (want.abs() + once) + 2.0 ** -10 * each).all())
                held_rows.append(got)
            for h in range(HEADS):
                k, v = (t[:, h // (HEADS // KV)] for t in held_rows)
                o, _, size, b = plain_attention(part[:, h], k, v, True, HD ** -0.5)
                held(out[start:start + n, h], (o, 2.0 ** -8 * o.abs() + (2.0 ** -10 + 2.0 ** -15 * b[:, None]) * size + 1e-30))
            start += n


@pytest.mark.parametrize("requests", [3, 40])
def test_captured(requests):
    """Replays of the captured step over a cache of its own give the bits of eager steps over another."""
    step, gen = Step(requests), torch.Generator().manual_seed(1)
    ones = torch.ones(requests, dtype=torch.int32, device="cuda")
    xs = [torch.randn(requests, WIDTH, generator=gen).bfloat16().cuda() for _ in range(4)]

    def run(x, cache):
        plan = cache.plan(ones, rows=requests, max_fresh=1)
        return step(x, (cache.length - 1).expand(3, requests).contiguous(), cache, plan)[-1]

    eager, kept = cache_of(requests, 64), cache_of(requests, 64)
    want = [run(x, eager).clone() for x in xs]
    x = xs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = run(x, kept)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(x, kept)
    for i in range(1, 4):
        x.copy_(xs[i])
        graph.replay()
        assert torch.equal(out, want[i])


def test_example_runs():
    path = pathlib.Path(__file__).resolve().parents[1] / "examples" / "w4_stream.py"
    spec = importlib.util.spec_from_file_location("w4_stream", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    assert math.isfinite(module.run(layers=1, requests=3, steps=4, say=lambda _: None))
