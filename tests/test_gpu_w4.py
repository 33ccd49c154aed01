"""GPU: products with 4-bit weights (``b200t2w.w4``) against a plain statement in 64 bits.  Codes, scales and zeros are read
back exactly; what products may be off by is derived in ``w4_ref``."""

import math

import pytest
import torch

import w4_ref as ref
from b200t2w import lib as L
from b200t2w import w4

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def _dev():
    assert torch.cuda.is_available()
    assert L.load().t2w_device_ok(torch.cuda.current_device()) == 1


def cuda(w):
    return tuple(None if t is None else t.cuda() for t in w)


def normal(gen, *size, dtype=BF16):
    return torch.randn(*size, generator=gen).to(dtype)


def held(out, want):
    y, lim = want
    d = (out.double().cpu() - y).abs()
    assert out.shape == y.shape and bool((d <= lim).all()), float((d / lim).max())


SHAPES = [  # rows, k, n
    (1, 32, 1), (1, 96, 5), (2, 128, 64), (3, 160, 63), (7, 1024, 200), (8, 256, 65), (9, 384, 129), (16, 2048, 64), (17, 544, 100),
    (31, 1024, 257), (33, 4096, 80), (64, 1152, 192), (65, 288, 130), (100, 640, 333), (128, 512, 128), (129, 1024, 512),
    (200, 96, 70), (257, 2048, 96), (300, 736, 1000), (513, 256, 264)]


@pytest.mark.parametrize("rows,k,n", SHAPES)
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True), (128, False)])
def test_linear(rows, k, n, group, zeros):
    group = group if k % group == 0 else 32
    gen = torch.Generator().manual_seed(rows * 7 + k + n)
    for i, (dtype, scale_dtype) in enumerate(((BF16, BF16), (FP16, FP16), (BF16, FP16), (FP16, BF16))):
        w = ref.weights(n, k, group, zeros, scale_dtype, gen)
        x = normal(gen, rows, k, dtype=dtype)
        bias = normal(gen, n, dtype=dtype) if i % 2 else None
        residual = normal(gen, rows, n, dtype=dtype) if i in (1, 2) else None
        p = w4.pack(*cuda(w))
        out = w4.linear(x.cuda(), p, *(None if t is None else t.cuda() for t in (bias, residual)))
        assert out.dtype == dtype
        held(out, ref.linear(x, w, bias, residual))
        p.check()


@pytest.mark.parametrize("rows,k,f", [(1, 32, 1), (2, 128, 32), (5, 160, 33), (8, 1024, 70), (9, 512, 8), (16, 96, 31), (40, 2048, 100),
                                      (64, 256, 129), (65, 1024, 64), (130, 384, 200), (260, 1152, 77), (300, 128, 65)])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_gated(rows, k, f, act):
    gen = torch.Generator().manual_seed(rows + k * 3 + f)
    for dtype, group, zeros in ((BF16, 128, False), (FP16, 64, True), (BF16, 32, True)):
        group = group if k % group == 0 else 32
        gate, up = (ref.weights(f, k, group, zeros, dtype, gen) for _ in range(2))
        x = normal(gen, rows, k, dtype=dtype)
        p = w4.pack_gated(cuda(gate), cuda(up))
        out = w4.gated(x.cuda(), p, act)
        held(out, ref.gated(x, gate, up, act))
        p.check()


@pytest.mark.parametrize("rows", [3, 40])
@pytest.mark.parametrize("act,gates", [("silu", (-80.0, -110.0, -0.5)), ("gelu_tanh", (-10.0, -11.5, -0.0625))])
def test_gated_far_below_zero(rows, act, gates):
    """Gate sums whose sigmoid is near the least fp32 numbers, where the activation is still more than bf16's.

    One product of each sum is not 0, so sums are exact.  Beside the relative error of ``w4_ref.gated``: GELU's argument s has
    four roundings, so that e^s is off by |s| 2^-22 of itself; a subnormal e^s and its product with g are off by a step,
    2^-149, each (twice that is allowed)."""
    g = torch.arange(*gates, dtype=torch.float64)
    n = g.numel()
    gate, up = (torch.full((8, 32), 8, dtype=torch.uint8) for _ in range(2))
    gate[:, 0] = up[:, 1] = 9
    one = torch.ones(8, 1, dtype=BF16)
    p = w4.pack_gated((gate.cuda(), one.cuda()), (up.cuda(), one.cuda()))
    for u in (1.0, -2.0 ** 20, 2.0 ** 60):
        for first in range(0, n, rows):
            part = g[first:first + rows]
            x = torch.zeros(rows, 32, dtype=BF16)
            x[:part.numel(), 0], x[:, 1] = part.to(BF16), u
            assert torch.equal(x[:part.numel(), 0].double(), part)
            v = x[:, :1].double()
            s = v if act == "silu" else 2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)
            a = v * torch.sigmoid(s)
            e = (8 + 3.2 * s.abs()) * 2.0 ** -23 * a.abs() + 2.0 ** -148 * (v.abs() + 1)
            y = (a * u).expand(rows, 8)
            held(w4.gated(x.cuda(), p, act), (y, ref.rounded(y, (e * abs(u) + 2.0 ** -24 * y.abs()).expand(rows, 8), BF16)))


@pytest.mark.parametrize("n,k,group,zeros,dtype", [(1, 32, 32, False, BF16), (65, 160, 32, True, FP16), (200, 384, 128, True, BF16),
                                                   (64, 128, 64, False, FP16), (130, 4096, 64, True, BF16)])
def test_pack_and_unpack(n, k, group, zeros, dtype):
    gen = torch.Generator().manual_seed(n + k)
    a, b = (ref.weights(n, k, group, zeros, dtype, gen) for _ in range(2))
    assert torch.equal(w4.pack(*cuda(a)).unpack().double().cpu(), ref.dense(a))
    p = w4.pack_gated(cuda(a), cuda(b))
    assert p.is_gated and p.zeros == zeros and p.scale_dtype == dtype
    for got, want in zip(p.unpack(), (a, b)):
        assert torch.equal(got.double().cpu(), ref.dense(want))
    # views: codes and scales as columns of wider matrices
    wide = torch.full((n, k + 24), 77, dtype=torch.uint8, device="cuda")
    wide[:, 8:8 + k] = a[0].cuda()
    s = torch.full((n, k // group + 3), float("nan"), dtype=dtype, device="cuda")
    s[:, 1:1 + k // group] = a[1].cuda()
    z = None if a[2] is None else a[2].cuda()
    assert torch.equal(w4.pack(wide[:, 8:8 + k], s[:, 1:1 + k // group], z).buffer, w4.pack(*cuda(a)).buffer)


@pytest.mark.parametrize("rows", [1, 8, 24, 150, 300])
def test_rows_that_are_not_finite_stay_to_themselves(rows):
    """A NaN or an infinity in one row of x reaches that row's outputs and no others; what lies between the rows of x is not
    read at all."""
    gen = torch.Generator().manual_seed(rows)
    k, n = 416, 150
    w = w4.pack(*cuda(ref.weights(n, k, 32, True, BF16, gen)))
    g = w4.pack_gated(*(cuda(ref.weights(n, k, 32, True, BF16, gen)) for _ in range(2)))
    wide = torch.full((rows, k + 40), float("nan"), dtype=BF16, device="cuda")
    x = wide[:, :k]
    x.copy_(normal(gen, rows, k))
    for f in (lambda: w4.linear(x, w), lambda: w4.gated(x, g)):
        want = f()
        assert bool(torch.isfinite(want).all())
        assert torch.equal(want, f())  # the same bits in every call
        bad = rows // 2
        keep = x[bad].clone()
        for v in (float("nan"), float("inf")):
            x[bad, 5] = v
            got = f()
            assert bool((~torch.isfinite(got[bad])).any())
            others = [i for i in range(rows) if i != bad]
            assert torch.equal(got[others], want[others])
            x[bad] = keep


@pytest.mark.parametrize("rows,k,n", [
    (1, 32, 40000), (8, 512, 20000),    # few rows: more row blocks than the clusters take in one pass, one and four tiles of k
    (3, 4096, 700), (16, 1056, 9000),   # a warp's tiles of two row blocks; two columns of blocks
    (20, 128, 39000), (33, 384, 20000),  # more rows: more tiles than blocks, with an odd number of row blocks
    (700, 192, 7000), (1025, 64, 5000)])
@pytest.mark.parametrize("group", [32, 64])
def test_many_row_blocks(rows, k, n, group):
    """Row blocks by the hundred, against the statement on the GPU."""
    group = group if k % group == 0 else 32
    gen = torch.Generator().manual_seed(rows + n)
    w = cuda(ref.weights(n, k, group, True, BF16, gen))
    x, bias = normal(gen, rows, k).cuda(), normal(gen, n).cuda()
    y, lim = ref.linear(x, w, bias)
    held(w4.linear(x, w4.pack(*w), bias), (y.cpu(), lim.cpu()))
    half = tuple(None if t is None else t[:n // 2] for t in w), tuple(None if t is None else t[n // 2:n // 2 * 2] for t in w)
    y, lim = ref.gated(x, *half, "silu")
    held(w4.gated(x, w4.pack_gated(*half)), (y.cpu(), lim.cpu()))


@pytest.mark.parametrize("rows", [2, 40, 130])
def test_offsets_past_32_bits(rows):
    """A weight of 4.6 GB: its last rows."""
    k, n = 65536, 131136
    gen = torch.Generator(device="cuda").manual_seed(rows)
    codes = torch.randint(0, 16, (n, k), generator=gen, device="cuda", dtype=torch.uint8)
    scales = (torch.rand(n, k // 128, generator=gen, device="cuda") * 0.01).to(BF16)
    p = w4.pack(codes, scales)
    assert p.buffer.numel() > 2 ** 32
    x = torch.randn(rows, k, generator=gen, device="cuda").to(BF16)
    out = w4.linear(x, p)
    for part in (slice(0, 40), slice(n - 100, n)):
        y, lim = ref.linear(x.cpu(), (codes[part].cpu(), scales[part].cpu(), None))
        held(out[:, part], (y, lim))


def test_strides_and_rows():
    gen = torch.Generator().manual_seed(3)
    k, n = 256, 72
    w = ref.weights(n, k, 64, False, BF16, gen)
    p = w4.pack(*cuda(w))
    x, r = normal(gen, 40, k), normal(gen, 40, n)
    res = torch.zeros(40, n + 5, dtype=BF16, device="cuda")
    res[:, 3:3 + n] = r.cuda()
    both = torch.zeros(40, 2, k, dtype=BF16, device="cuda")
    both[:, 1] = x.cuda()
    held(w4.linear(both[:, 1], p, residual=res[:, 3:3 + n]), ref.linear(x, w, None, r))
    every = both.view(20, 4, k)[:, 3]  # every other row
    held(w4.linear(every, p), ref.linear(x[1::2], w))
    assert w4.linear(x[:0].cuda(), p).shape == (0, n)
    one = torch.zeros(1, k + 3, dtype=BF16, device="cuda")[:, :k]  # a pitch is of no account where there is one row
    assert w4.linear(one, p).shape == (1, n)


def test_extremes():
    """Largest codes and zeros of either sign, scales from the smallest to large ones, groups with scale 0."""
    k, n = 256, 64
    gen = torch.Generator().manual_seed(5)
    codes = torch.zeros(n, k, dtype=torch.uint8)
    codes[1::2] = 15
    zeros = torch.zeros(n, 2, dtype=torch.uint8)
    zeros[::2] = 15
    for dtype in (BF16, FP16):
        scales = torch.exp2(torch.linspace(-24, 10, n)).to(dtype)[:, None].repeat(1, 2)
        scales[7] = 0
        x = (normal(gen, 3, k).float() * torch.tensor([[2.0 ** -14], [1.0], [8.0]])).to(dtype)
        w = (codes, scales, zeros)
        y, lim = ref.linear(x, w)
        out = w4.linear(x.cuda(), w4.pack(*cuda(w))).double().cpu()
        top = torch.finfo(dtype).max
        over = y.abs() > 0.99 * top
        assert bool(((out - y).abs() <= lim)[~over].all())
        assert bool((out[:, 7] == 0).all())


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("zeros", [False, True])
def test_quantize_and_products(dtype, zeros):
    gen = torch.Generator().manual_seed(11)
    m = normal(gen, 96, 512, dtype=dtype)
    codes, scales, z = w4.quantize(m.cuda(), 64, zeros)
    cpu = w4.quantize(m, 64, zeros)
    for a, b in zip((codes, scales, z), cpu):
        assert (a is None and b is None) or torch.equal(a.cpu(), b)
    x = normal(gen, 4, 512, dtype=dtype)
    held(w4.linear(x.cuda(), w4.pack(codes, scales, z)), ref.linear(x, cpu))


@pytest.mark.parametrize("rows", [1, 40])
def test_feed_forward(rows):
    gen = torch.Generator().manual_seed(2)
    k, f = 512, 1000 // 32 * 32
    gate, up, down = (ref.weights(a, b, 32, True, BF16, gen) for a, b in ((f, k), (f, k), (k, f)))
    x, r = normal(gen, rows, k), normal(gen, rows, k)
    gu, d = w4.pack_gated(cuda(gate), cuda(up)), w4.pack(*cuda(down))
    out = w4.feed_forward(x.cuda(), gu, d, residual=r.cuda())
    h = w4.gated(x.cuda(), gu)
    assert torch.equal(out, w4.linear(h, d, residual=r.cuda()))
    held(out, ref.linear(h.cpu(), down, None, r))


@pytest.mark.parametrize("rows", [1, 12, 200])
def test_captured_and_on_other_streams(rows):
    """Two graphs over one weight, replayed on two streams at once, and an eager call beside them, give the bits that
    calls of their own give."""
    gen = torch.Generator().manual_seed(rows)
    k, f = 1024, 512
    gu = w4.pack_gated(*(cuda(ref.weights(f, k, 128, False, BF16, gen)) for _ in range(2)))
    down = w4.pack(*cuda(ref.weights(k, f, 128, True, BF16, gen)))
    xs = [normal(gen, rows, k).cuda() for _ in range(3)]
    want = [w4.feed_forward(x, gu, down, residual=x) for x in xs]
    torch.cuda.synchronize()
    streams, graphs, held_in, outs = [torch.cuda.Stream() for _ in range(2)], [], [], []
    for i in range(2):
        buf = torch.zeros_like(xs[0])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = buf
            for _ in range(3):
                y = w4.feed_forward(buf, gu, down, residual=buf)
        graphs.append(graph)
        held_in.append(buf)
        outs.append(y)
    torch.cuda.synchronize()
    for _ in range(3):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                held_in[i].copy_(xs[i])
                graphs[i].replay()
        eager = w4.feed_forward(xs[2], gu, down, residual=xs[2])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[2])
    gu.check()
    down.check()


@pytest.mark.parametrize("rows", [2, 40])
def test_a_status_is_told_once(rows):
    """A status as a wait that gave up records it is raised by one ``check``, and products after it are judged by themselves."""
    gen = torch.Generator().manual_seed(7)
    w, x = ref.weights(80, 160, 32, True, BF16, gen), normal(gen, rows, 160)
    p = w4.pack(*cuda(w))
    laid_out = p.buffer.clone()
    p.buffer[:4].view(torch.int32).fill_(-4)
    torch.cuda.synchronize()
    with pytest.raises(L.T2WError) as e:
        p.check()
    assert e.value.status == -4
    p.check()
    out = w4.linear(x.cuda(), p)
    p.check()
    held(out, ref.linear(x, w))
    assert torch.equal(p.buffer, laid_out)


def test_refusals():
    gen = torch.Generator().manual_seed(1)
    w = ref.weights(64, 128, 64, True, BF16, gen)
    p = w4.pack(*cuda(w))
    g = w4.pack_gated(cuda(w), cuda(w))
    x = normal(gen, 4, 128).cuda()
    wide = torch.zeros(4, 132, dtype=BF16, device="cuda")
    bad = [
        lambda: w4.linear(x.float(), p), lambda: w4.linear(x.cpu(), p), lambda: w4.linear(x[:, :64], p), lambda: w4.linear(x[0], p),
        lambda: w4.linear(wide[:, :128], p), lambda: w4.linear(wide.view(-1)[4:516].view(4, 128), p),
        lambda: w4.linear(torch.zeros(128, 8, dtype=BF16, device="cuda").T, p),
        lambda: w4.linear(x[:1].expand(4, 128), p), lambda: w4.linear(x, g), lambda: w4.gated(x, p),
        lambda: w4.linear(x, p, bias=torch.zeros(63, dtype=BF16, device="cuda")),
        lambda: w4.linear(x, p, bias=torch.zeros(64, device="cuda")),
        lambda: w4.linear(x, p, residual=torch.zeros(4, 64, dtype=FP16, device="cuda")),
        lambda: w4.linear(x, p, residual=torch.zeros(3, 64, dtype=BF16, device="cuda")),
        lambda: w4.linear(x, p, residual=torch.zeros(64, 4, dtype=BF16, device="cuda").T),
        lambda: w4.linear(x, p, residual=torch.zeros(4, 64, dtype=BF16)),
        lambda: w4.linear(x.clone().requires_grad_(), p),
        lambda: w4.linear(x, w4.Weight4(p.buffer[:-16], p.n, p.k, p.group, p.kind)),
        lambda: w4.linear(x, w4.Weight4(p.buffer, p.n, p.k, 128, p.kind)),
    ]
    for f in bad:
        with pytest.raises(RuntimeError):
            f()
    for kw in (dict(n=0), dict(k=120), dict(group=48), dict(n=-5)):
        a = dict(n=p.n, k=p.k, group=p.group) | kw
        with pytest.raises((L.T2WError, RuntimeError)):
            w4.linear(x, w4.Weight4(p.buffer, a["n"], a["k"], a["group"], p.kind))
    with pytest.raises(ValueError):
        w4.gated(x, g, act="relu")
    with torch.no_grad():
        w4.linear(x.clone().requires_grad_(), p)
    assert bool(torch.isfinite(w4.linear(x, p)).all())  # and the library goes on


def test_bias_and_residual_that_want_a_gradient():
    """The products have no gradient: what would have to get one is refused where gradients are recorded."""
    gen = torch.Generator().manual_seed(4)
    w = ref.weights(64, 128, 64, True, BF16, gen)
    p = w4.pack(*cuda(w))
    x, r, b = normal(gen, 4, 128), normal(gen, 4, 64), normal(gen, 64)
    xs, rs, bs = x.cuda(), r.cuda().requires_grad_(), torch.nn.Parameter(b.cuda())
    for kw in (dict(bias=bs), dict(residual=rs), dict(bias=bs.detach(), residual=rs), dict(bias=bs, residual=rs.detach())):
        with pytest.raises(RuntimeError, match="no gradient"):
            w4.linear(xs, p, **kw)
    with pytest.raises(RuntimeError, match="no gradient"):
        w4.feed_forward(xs, w4.pack_gated(cuda(w), cuda(w)), w4.pack(*cuda(ref.weights(64, 64, 64, True, BF16, gen))), residual=rs)
    with torch.no_grad():
        out = w4.linear(xs, p, bs, rs)
    assert not out.requires_grad
    held(out, ref.linear(x, w, b, r))


def test_weights_that_cannot_be_packed():
    gen = torch.Generator().manual_seed(1)
    codes, scales, zeros = cuda(ref.weights(64, 128, 64, True, BF16, gen))
    big = codes.clone()
    big[3, 4] = 16
    nan = scales.clone()
    nan[0, 0] = float("nan")
    for args in ((big, scales, zeros), (codes, scales, zeros + 16), (codes, nan, zeros), (codes, scales.float(), zeros),
                 (codes.int(), scales, zeros), (codes, scales[:32], zeros), (codes[:, :120], scales, zeros), (codes[0], scales, zeros)):
        with pytest.raises(ValueError):
            w4.pack(*args)
    for args in ((codes, scales, zeros[:5]), (codes, scales.cpu(), zeros), (codes.T.contiguous().T, scales, zeros)):
        with pytest.raises(RuntimeError):
            w4.pack(*args)
    with pytest.raises(ValueError):
        w4.pack_gated((codes, scales, zeros), (codes, scales, None))
    with pytest.raises(ValueError):
        w4.pack_gated((codes, scales, zeros), (codes[:32], scales[:32], zeros[:32]))


@pytest.mark.skipif(not torch.cuda.is_available() or torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_another_device():
    gen = torch.Generator().manual_seed(9)
    w, x = ref.weights(100, 256, 64, True, BF16, gen), normal(gen, 5, 256)
    with torch.cuda.device(0):
        p = w4.pack(*(t.to("cuda:1") for t in w))
        held(w4.linear(x.to("cuda:1"), p), ref.linear(x, w))
        with pytest.raises(RuntimeError):
            w4.linear(x.to("cuda:0"), p)
