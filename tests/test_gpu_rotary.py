"""GPU: rotary positions with several axes (``b200t2w.rotary``) against a plain statement in 64 bits.

An output may be off by half a step of its type, plus 2^-21 (|x| + |y|) for its pair (x, y): a sine and a cosine of the angle's leading
32 bits (2^-32 of a turn, 2^-29 radians) converted to fp32 (2^-24 of at most pi radians, 2^-22), the functions' own error (2
steps, 2^-23), and two products and a sum (2 * 2^-24 of both)."""

import pytest
import torch

import w4_ref as ref
from b200t2w import lib as L
from b200t2w.rotary import Rotary

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def _dev():
    assert torch.cuda.is_available()
    assert L.load().t2w_device_ok(torch.cuda.current_device()) == 1


def inv_freq(rot, base):
    return torch.tensor([base ** (-2 * i / rot) for i in range(rot // 2)], dtype=torch.float64)


def axis_of(sections):
    return torch.tensor([a for a, s in enumerate(sections) for _ in range(s)])


def held(out, x, positions, axis, freq, rot, adjacent, inverse):
    y = ref.turned(x, positions, axis, freq, rot, adjacent, inverse)
    d = x.double()
    size = torch.zeros_like(d)
    if adjacent:
        size[..., :rot] = (d[..., 0:rot:2].abs() + d[..., 1:rot:2].abs()).repeat_interleave(2, -1)
    else:
        size[..., :rot] = (d[..., :rot // 2].abs() + d[..., rot // 2:rot].abs()).repeat(1, 1, 2)
    # a frequency is off by 2^-53 in the statement itself
    e = (2.0 ** -21 + positions.abs().max().double() * 2.0 ** -52) * size
    lim = ref.rounded(y, e, x.dtype)
    lim[..., rot:] = 0  # kept as they are
    got = out.double().cpu()
    assert out.shape == x.shape and bool(((got - y).abs() <= lim).all()), float(((got - y).abs() / lim.clamp(min=1e-300)).max())


@pytest.mark.parametrize("hd,rot,sections", [(64, 64, [32]), (128, 128, [16, 24, 24]), (80, 80, [20, 20]), (128, 32, [4, 4, 4, 4]),
                                             (16, 16, [8]), (256, 128, [64, 0]), (96, 48, [0, 7, 17]), (24, 16, [1, 2, 5])])
@pytest.mark.parametrize("adjacent", [False, True])
def test_turns(hd, rot, sections, adjacent):
    gen = torch.Generator().manual_seed(hd + rot)
    turn = Rotary(hd, sections, base=10000.0, rotary_dim=rot, pairs="adjacent" if adjacent else "half")
    freq, axis = inv_freq(rot, 10000.0), axis_of(sections)
    for rows, heads, kv, dtype, wide, far, inverse in ((1, 8, 2, BF16, False, 100, False), (7, 3, 1, FP16, True, 5000, False),
                                                       (130, 32, 8, BF16, True, 1000000, True), (65, 1, 1, FP16, False, 70, True),
                                                       (33, 40, 40, BF16, False, 300000, False)):
        pos = torch.randint(-far // 10, far, (len(sections), rows), generator=gen, dtype=torch.int64 if wide else torch.int32)
        qkv = torch.randn(rows, heads + 2 * kv, hd, generator=gen).to(dtype)
        q, k = qkv[:, :heads], qkv[:, heads:heads + kv]
        dev = qkv.cuda()
        before = dev.clone()
        a, b = turn(dev[:, :heads], dev[:, heads:heads + kv], pos.cuda(), inverse=inverse)
        assert a.is_contiguous() and b.is_contiguous() and torch.equal(dev, before)
        held(a, q, pos, axis, freq, rot, adjacent, inverse)
        held(b, k, pos, axis, freq, rot, adjacent, inverse)
        # in place: the same bits, and the values that lie between them as they were
        turn.apply_(dev[:, :heads], dev[:, heads:heads + kv], pos.cuda(), inverse=inverse)
        assert torch.equal(dev[:, :heads], a) and torch.equal(dev[:, heads:heads + kv], b)
        assert torch.equal(dev[:, heads + kv:], before[:, heads + kv:])
        alone, none = turn(q.cuda(), None, pos.cuda(), inverse=inverse)
        assert none is None and torch.equal(alone, a)


def test_far_positions():
    """As exact at 2^31 as at 1: whole positions times fixed-point frequencies, here against integers of any size."""
    import decimal

    hd, base = 128, 1000000.0
    turn = Rotary(hd, base=base)
    pos = [2 ** 31 - 1, -2 ** 31, 2 ** 30 + 12345, 1, 0, -1]
    one = torch.zeros(len(pos), 1, hd, dtype=FP16)
    one[:, :, :64] = 1
    got, _ = turn(one.cuda(), None, torch.tensor(pos, dtype=torch.int32).cuda())
    with decimal.localcontext() as c:
        c.prec = 50
        two_pi = decimal.Decimal("6.2831853071795864769252867665590057683943387987502")
        angle = [[float((p * (decimal.Decimal(base).ln() * (-2 * i) / hd).exp()) % two_pi) for i in range(64)] for p in pos]
    angle = torch.tensor(angle, dtype=torch.float64)
    want = torch.cat([torch.cos(angle), torch.sin(angle)], 1)
    d = (got[:, 0].double().cpu() - want).abs()
    assert bool((d <= 2.0 ** -11 * want.abs() + 2.0 ** -21 + 2.0 ** -24).all()), float(d.max())


def test_interleaved_sections_and_own_frequencies():
    gen = torch.Generator().manual_seed(4)
    x = torch.randn(20, 2, 64, generator=gen).to(FP16)
    pos = torch.randint(0, 900, (3, 20), generator=gen)
    turn = Rotary(64, [14, 9, 9], interleaved=True)
    axis = torch.tensor([i % 3 if i < 27 else 0 for i in range(32)])
    held(turn(x.cuda(), None, pos.cuda())[0], x, pos, axis, inv_freq(64, 10000.0), 64, False, False)
    own = torch.rand(32, generator=gen, dtype=torch.float64) * 2 - 1
    own[3], own[4] = 0.0, 7.5
    turn = Rotary(64, [14, 9, 9], inv_freq=own)
    held(turn(x.cuda(), None, pos.cuda())[0], x, pos, axis_of([14, 9, 9]), own, 64, False, False)


@pytest.mark.parametrize("adjacent", [False, True])
def test_frequencies_that_start_again(adjacent):
    """Height and width with a ladder of their own each, as image towers have them, given as own frequencies."""
    gen = torch.Generator().manual_seed(5)
    rot, x = 80, torch.randn(30, 2, 80, generator=gen).to(BF16)
    pos = torch.randint(0, 70, (2, 30), generator=gen)
    turn = Rotary(rot, [20, 20], pairs="adjacent" if adjacent else "half",
                  inv_freq=2 * [10000.0 ** (-4 * i / rot) for i in range(rot // 4)])
    held(turn(x.cuda(), None, pos.cuda())[0], x, pos, axis_of([20, 20]), torch.cat([inv_freq(rot // 2, 10000.0)] * 2), rot, adjacent, False)


def test_inverse_is_the_gradient():
    """With L = sum w . turned(x): the gradient is the inverse turn of w, against the formula's (autograd in 64 bits) and
    against differences of L."""
    gen = torch.Generator().manual_seed(6)
    pos = torch.randint(0, 4000, (2, 5), generator=gen)
    for adjacent in (False, True):
        turn = Rotary(32, [10, 6], pairs="adjacent" if adjacent else "half")
        freq, axis = inv_freq(32, 10000.0), axis_of([10, 6])
        w = torch.randn(5, 3, 32, generator=gen).to(FP16)
        x = torch.randn(5, 3, 32, generator=gen, dtype=torch.float64, requires_grad=True)

        def loss(v):
            angle = pos.double()[axis] * freq[:, None]
            c, s = torch.cos(angle).T[:, None], torch.sin(angle).T[:, None]
            a, b = (v[..., 0::2], v[..., 1::2]) if adjacent else (v[..., :16], v[..., 16:])
            p, q = (w[..., 0::2], w[..., 1::2]) if adjacent else (w[..., :16], w[..., 16:])
            return ((a * c - b * s) * p.double() + (b * c + a * s) * q.double()).sum()

        want, = torch.autograd.grad(loss(x), x)
        got = turn(w.cuda(), None, pos.cuda(), inverse=True)[0].double().cpu()
        lim = 2.0 ** -11 * want.abs() + 2.0 ** -20 * 8
        assert bool(((got - want).abs() <= lim).all())
        v = x.detach()
        for _ in range(8):
            r, h, i = (int(torch.randint(0, m, (1,), generator=gen)) for m in (5, 3, 32))
            e = torch.zeros_like(v)
            e[r, h, i] = 0.5
            assert abs(float(loss(v + e) - loss(v - e)) - float(got[r, h, i])) <= float(lim[r, h, i]) + 1e-9  # L is linear


def test_rows_heads_and_strides():
    gen = torch.Generator().manual_seed(8)
    turn = Rotary(64, [32])
    freq, axis = inv_freq(64, 10000.0), axis_of([32])
    pos = torch.randint(0, 900, (12,), generator=gen, dtype=torch.int32)
    x = torch.randn(12, 4, 64, generator=gen).to(BF16)
    by_head = x.transpose(0, 1).contiguous().cuda().transpose(0, 1)  # [heads][rows] in memory
    held(turn(by_head, None, pos.cuda())[0], x, pos[None], axis, freq, 64, False, False)
    want = turn(x.cuda(), None, pos.cuda())[0]
    turn.apply_(by_head, None, pos.cuda())
    assert torch.equal(by_head, want)
    same = x[:1].cuda().expand(12, 4, 64)  # one row, turned to twelve places
    held(turn(same, None, pos.cuda())[0], x[:1].expand(12, 4, 64), pos[None], axis, freq, 64, False, False)
    assert turn(x[:0].cuda(), x[:0].cuda(), pos[:0].cuda())[1].shape == (0, 4, 64)
    e = turn(x.cuda(), x[:, :0].cuda(), pos.cuda())
    assert torch.equal(e[0], want) and e[1].shape == (12, 0, 64)
    # a value that is not finite reaches its own pair alone
    bad = x.clone()
    bad[3, 2, 5] = float("nan")
    got = turn(bad.cuda(), None, pos.cuda())[0]
    hit = torch.zeros(12, 4, 64, dtype=torch.bool)
    hit[3, 2, 5] = hit[3, 2, 37] = True
    assert torch.equal(torch.isnan(got).cpu(), hit) and torch.equal(got.cpu()[~hit], want.cpu()[~hit])


@pytest.mark.parametrize("rows", [1, 2, 70])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_one_line_of_positions_for_all_axes(rows, dtype):
    gen = torch.Generator().manual_seed(rows)
    turn = Rotary(64, [12, 10, 10])
    x = torch.randn(rows, 4, 64, generator=gen).to(BF16)
    line = torch.randint(0, 90000, (rows,), generator=gen, dtype=dtype)
    q, pos = x.cuda(), line.cuda().expand(3, rows)
    assert pos.stride(0) == 0
    want = turn(q, None, pos.contiguous())[0]
    assert torch.equal(turn(q, None, pos)[0], want)
    held(want, x, line.expand(3, rows), axis_of([12, 10, 10]), inv_freq(64, 10000.0), 64, False, False)
    turn.apply_(q, None, pos)
    assert torch.equal(q, want)


@pytest.mark.parametrize("rows", [1, 5])
def test_heads_of_q_and_k_in_turn(rows):
    """In place in rows [heads, 3, head_dim], where q's and k's heads alternate and share nothing; and strided heads that do."""
    gen = torch.Generator().manual_seed(rows)
    turn = Rotary(64, [16, 16])
    pos = torch.randint(0, 900, (2, rows), generator=gen).cuda()
    x = torch.randn(rows, 8, 3, 64, generator=gen).to(BF16).cuda()
    a, b = turn(x[:, :, 0], x[:, :, 1], pos)
    y = x.clone()
    turn.apply_(y[:, :, 0], y[:, :, 1], pos)
    assert torch.equal(y[:, :, 0], a) and torch.equal(y[:, :, 1], b) and torch.equal(y[:, :, 2], x[:, :, 2])
    y = x.clone()
    turn.apply_(y[:, :, 2], y[:, 1:5, 0], pos)
    assert torch.equal(y[:, :, 2], turn(x[:, :, 2], None, pos)[0]) and torch.equal(y[:, 1:5, 0], a[:, 1:5])
    assert torch.equal(y[:, :, 1], x[:, :, 1]) and torch.equal(y[:, 5:, 0], x[:, 5:, 0])
    for off in (8, 56, 3 * 64 + 8, 2 * 64 + 8):  # a part of a head in common
        k = y.view(-1).as_strided((rows, 5, 64), (8 * 3 * 64, 3 * 64, 1), off)
        with pytest.raises(L.T2WError):
            turn.apply_(y[:, :, 0], k, pos)


def test_as_many_rows_as_there_may_be():
    """2^31 - 1 rows of one head: the first and the last ones, in place."""
    rows, hd = 2 ** 31 - 1, 16
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 90 << 30:
        pytest.skip("needs 77 GB of GPU memory")
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(600, 1, hd, generator=gen).to(BF16)
    pos = torch.randint(0, 5000, (600,), generator=gen, dtype=torch.int32)
    q = torch.zeros(rows, 1, hd, dtype=BF16, device="cuda")
    p = torch.zeros(rows, dtype=torch.int32, device="cuda")
    q[:300], q[-300:], p[:300], p[-300:] = x[:300].cuda(), x[300:].cuda(), pos[:300].cuda(), pos[300:].cuda()
    Rotary(hd).apply_(q, None, p)
    held(torch.cat([q[:300], q[-300:]]), x, pos[None], axis_of([hd // 2]), inv_freq(hd, 10000.0), hd, False, False)
    assert not bool(q[300:1000].any()) and not bool(q[-1000:-300].any())
    del q, p
    torch.cuda.empty_cache()


def test_captured():
    gen = torch.Generator().manual_seed(8)
    turn = Rotary(128, [16, 24, 24])
    q, k = torch.randn(9, 8, 128, generator=gen).to(BF16).cuda(), torch.randn(9, 2, 128, generator=gen).to(BF16).cuda()
    pos = torch.zeros(3, 9, dtype=torch.int32, device="cuda")
    turn(q, k, pos)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = turn(q, k, pos)
    for i in range(3):
        pos.copy_(torch.randint(0, 5000, (3, 9), generator=gen))
        graph.replay()
        c, d = turn(q, k, pos)
        assert torch.equal(a, c) and torch.equal(b, d)


def test_refusals():
    turn = Rotary(64, [16, 16])
    q, k = torch.zeros(4, 8, 64, dtype=BF16, device="cuda"), torch.zeros(4, 2, 64, dtype=BF16, device="cuda")
    pos = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    odd = torch.zeros(4 * 8 * 64 + 4, dtype=BF16, device="cuda")
    for f in (lambda: turn(q.float(), k, pos), lambda: turn(q, k.half(), pos), lambda: turn(q, k[:3], pos), lambda: turn(q, k, pos[:1]),
              lambda: turn(q, k, pos[0]), lambda: turn(q, k, pos.float()), lambda: turn(q, k, pos.cpu()), lambda: turn(q.cpu(), None, pos),
              lambda: turn(q, k, pos[:, :3]), lambda: turn(q[0], None, pos), lambda: turn(odd[4:].view(4, 8, 64), None, pos),
              lambda: turn(q.transpose(0, 1), k, pos), lambda: turn(q, k, pos.T.contiguous().T),
              lambda: turn.apply_(q[:1].expand(4, 8, 64), None, pos), lambda: turn.apply_(q[:, :1].expand(4, 8, 64), None, pos),
              lambda: turn.apply_(q, q, pos), lambda: turn(q.clone().requires_grad_(), k, pos)):
        with pytest.raises(RuntimeError):
            f()
    rows = torch.zeros(4, 12, 64, dtype=BF16, device="cuda")  # columns of the same rows: apart, and one head in both
    turn.apply_(rows[:, :8], rows[:, 8:10], pos)
    turn.apply_(rows[:, 4:], rows[:, :4], pos)
    for a, b in ((rows[:, :8], rows[:, 7:9]), (rows[:, 4:], rows[:, 3:5]), (rows[1:, :8], rows[:3, 7:])):
        with pytest.raises(L.T2WError):
            turn.apply_(a, b, pos[:, :a.shape[0]])
    with pytest.raises(ValueError):
        turn(q[..., :32], None, pos)
    turn(q, k, pos)


@pytest.mark.skipif(not torch.cuda.is_available() or torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_another_device():
    turn = Rotary(64, device="cuda:1")
    x = torch.randn(3, 2, 64).to(BF16)
    pos = torch.tensor([1, 2, 3])
    with torch.cuda.device(0):
        held(turn(x.to("cuda:1"), None, pos.to("cuda:1"))[0], x, pos[None], axis_of([32]), inv_freq(64, 10000.0), 64, False, False)
        with pytest.raises(RuntimeError):
            turn(x.to("cuda:0"), None, pos.to("cuda:0"))
