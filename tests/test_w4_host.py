"""CPU: quantising to 4 bits, the sizes and arguments that the products with 4-bit weights and the rotary positions take
and refuse, the rotary table.  No GPU work is enqueued here."""

import ctypes
import decimal
import math

import pytest
import torch

from b200t2w import lib as L
from b200t2w import w4
from b200t2w.rotary import Rotary

INVALID, UNSUPPORTED = -1, -5
BF16, FP16 = torch.bfloat16, torch.float16


def test_bytes():
    size = L.load().t2w_w4_bytes
    # a header of 128 bytes, then for 64 rows x 128 inputs 4096 bytes of codes and 2 (3 with zeros) a row and group
    assert size(64, 128, 128, 0, 0) == 128 + 4096 + 128
    assert size(64, 128, 32, 1, 0) == 128 + 4096 + 4 * 64 * 3
    assert size(65, 160, 32, 0, 0) == 128 + 4 * (4096 + 4 * 64 * 2)
    assert size(32, 128, 64, 0, 1) == size(64, 128, 64, 0, 0)  # a pair of 32 rows each
    assert size(33, 128, 64, 0, 1) == size(80, 128, 64, 0, 0)
    assert size(1 << 20, 1 << 16, 128, 0, 0) > 1 << 35
    for n, k, g in ((0, 128, 128), (-1, 128, 128), (1, 0, 32), (1, 128, 48), (1, 96, 64), (1, 128, 256), (1, 120, 32), (1, -128, 128),
                    (1, (1 << 24) + 128, 128), ((1 << 30) + 1, 32, 32)):
        assert size(n, k, g, 0, 0) == INVALID


def test_no_arguments():
    lib = L.load()
    assert lib.t2w_w4_linear(None, None) == INVALID and lib.t2w_rotary(None, None) == INVALID
    assert lib.t2w_w4_linear(ctypes.byref(L.W4LinearArgs()), None) == INVALID
    assert lib.t2w_w4_pack(None, None, None, None) == INVALID
    assert lib.t2w_w4_pack(ctypes.byref(L.W4Weight()), ctypes.byref(L.W4Source()), None, None) == INVALID
    assert lib.t2w_w4_unpack(ctypes.byref(L.W4Weight()), None, 0, None, 0, None) == INVALID
    assert lib.t2w_w4_status(None, None) == INVALID
    assert lib.t2w_rotary(ctypes.byref(L.RotaryArgs()), None) < 0


def linear_args(**kw):
    w = dict(n=64, k=128, group=64, scale_dtype=0, zeros=0, gated=0, buffer=1 << 20)
    a = dict(rows=4, dtype=0, act=0, x=1 << 20, x_ld=128, bias=None, residual=None, res_ld=0, out=1 << 20)
    for key, v in kw.items():
        (w if key in w else a)[key] = v
    return L.W4LinearArgs(w=L.W4Weight(**w), **a)


@pytest.mark.parametrize("kw,status", [
    (dict(rows=-1), INVALID), (dict(dtype=2), UNSUPPORTED), (dict(x=None), INVALID), (dict(out=None), INVALID),
    (dict(x=(1 << 20) + 8), INVALID), (dict(x_ld=132), INVALID), (dict(x_ld=120), INVALID), (dict(buffer=(1 << 20) + 64), INVALID),
    (dict(buffer=None), INVALID), (dict(scale_dtype=5), INVALID), (dict(group=16), INVALID), (dict(gated=1, act=3), INVALID),
    (dict(gated=1, bias=1 << 20), INVALID), (dict(gated=1, residual=1 << 20, res_ld=64), INVALID),
    (dict(residual=1 << 20, res_ld=63), INVALID), (dict(out=(1 << 20) + 1), INVALID)])
def test_products_that_there_are_not(kw, status):
    assert L.load().t2w_w4_linear(ctypes.byref(linear_args(**kw)), None) == status


@pytest.mark.parametrize("kw", [dict(bias=(1 << 20) + 1), dict(residual=(1 << 20) + 1, res_ld=64)])
def test_values_that_lie_between_two_addresses(kw):
    assert L.load().t2w_w4_linear(ctypes.byref(linear_args(**kw)), None) == INVALID
    assert L.load().t2w_w4_linear(ctypes.byref(linear_args(rows=40, **kw)), None) == INVALID


@pytest.mark.parametrize("gated", [0, 1])
def test_layouts_that_there_are_not(gated):
    lib, at = L.load(), 1 << 20
    w = L.W4Weight(n=64, k=128, group=64, scale_dtype=0, zeros=1, gated=gated, buffer=at)
    good = dict(codes=at, scales=at, zeros=at, code_ld=128, scale_ld=2, zero_ld=2)
    for kw in (dict(codes=None), dict(scales=None), dict(scales=at + 1), dict(zeros=None)):
        bad = ctypes.byref(L.W4Source(**(good | kw)))
        assert lib.t2w_w4_pack(ctypes.byref(w), bad, ctypes.byref(L.W4Source(**good)), None) == INVALID
        if gated:
            assert lib.t2w_w4_pack(ctypes.byref(w), ctypes.byref(L.W4Source(**good)), bad, None) == INVALID
    for out, ld in ((None, 128), (at + 2, 128), (at, 127), (at, 0), (at, -128)):
        assert lib.t2w_w4_unpack(ctypes.byref(w), out, ld, at, 128, None) == INVALID
        if gated:
            assert lib.t2w_w4_unpack(ctypes.byref(w), at, 128, out, ld, None) == INVALID


def test_no_rows_are_no_work():
    assert L.load().t2w_w4_linear(ctypes.byref(linear_args(rows=0, x=None, out=None)), None) == 0


def rotary_args(**kw):
    rows = dict(out=1 << 21, in_row_ld=512, in_head_ld=64, out_row_ld=512, out_head_ld=64)
    q, k = dict(rows), dict(rows, out=1 << 22)
    a = dict(rows=4, q_heads=8, k_heads=8, head_dim=64, rotary_dim=64, axes=2, adjacent=0, inverse=0, wide_positions=0, dtype=0,
             positions=1 << 20, pos_ld=4, table=1 << 20)
    src = 1 << 20
    for key, v in kw.items():
        if key == "q_in":
            src = v
        elif key.startswith("q_") and key != "q_heads":
            q[key[2:]] = v
        else:
            a[key] = v
    qs, ks = L.RotaryRows(**q), L.RotaryRows(**k)
    setattr(qs, "in", src)
    setattr(ks, "in", 1 << 19)
    return L.RotaryArgs(q=qs, k=ks, **a)


@pytest.mark.parametrize("kw,status", [
    (dict(rows=-1), INVALID), (dict(q_heads=-1), INVALID), (dict(head_dim=60), INVALID), (dict(rotary_dim=24), INVALID),
    (dict(rotary_dim=0), INVALID), (dict(rotary_dim=80), INVALID), (dict(axes=0), INVALID), (dict(dtype=9), UNSUPPORTED),
    (dict(positions=None), INVALID), (dict(table=None), INVALID), (dict(pos_ld=3), INVALID), (dict(q_in=None), INVALID),
    (dict(q_in=(1 << 20) + 8), INVALID), (dict(q_in_row_ld=516), INVALID), (dict(q_out=(1 << 21) + 2), INVALID),
    (dict(q_out_row_ld=64), INVALID), (dict(q_out_head_ld=0), INVALID), (dict(q_out=1 << 20, q_out_row_ld=1024), INVALID),
    (dict(q_out=1 << 22), INVALID), (dict(q_out=(1 << 22) - 64), INVALID), (dict(q_out=(1 << 22) + 2 * 512 + 128), INVALID),
    (dict(rows=1, pos_ld=1, axes=1, q_out=(1 << 22) + 128), INVALID), (dict(q_heads=20000, q_in_head_ld=64, q_out_row_ld=64 * 20000), UNSUPPORTED)])
def test_turns_that_there_are_not(kw, status):
    assert L.load().t2w_rotary(ctypes.byref(rotary_args(**kw)), None) == status


@pytest.mark.parametrize("rows,pos_ld,status", [(4, 0, UNSUPPORTED), (1, 0, UNSUPPORTED), (4, 4, UNSUPPORTED), (4, 1, INVALID),
                                                (4, -4, INVALID)])
def test_pitches_of_positions(rows, pos_ld, status):
    """0 is one line for all axes.  (20000 heads are more than the kernel has: what is not refused for its pitch is refused next.)"""
    kw = dict(rows=rows, pos_ld=pos_ld, q_heads=20000, q_in_head_ld=64, q_out_row_ld=64 * 20000, q_out=1 << 23)
    assert L.load().t2w_rotary(ctypes.byref(rotary_args(**kw)), None) == status


@pytest.mark.parametrize("off,wide,status", [(2, 0, INVALID), (4, 0, UNSUPPORTED), (4, 1, INVALID), (8, 1, UNSUPPORTED)])
def test_positions_that_lie_between_two_addresses(off, wide, status):
    kw = dict(positions=(1 << 20) + off, wide_positions=wide, q_heads=20000, q_in_head_ld=64, q_out_row_ld=64 * 20000)
    assert L.load().t2w_rotary(ctypes.byref(rotary_args(**kw)), None) == status


def test_rows_that_meet():
    """q and k in place at one row pitch are refused exactly where they have a value in common, heads that alternate among
    them.  Heads of 4112 values are more than the kernel has, so that a call that is not refused for this is refused next."""
    gen = torch.Generator().manual_seed(3)

    def pick(*of):
        return of[int(torch.randint(0, len(of), (1,), generator=gen))]

    hd, seen = 4112, {True: 0, False: 0}
    for _ in range(3000):
        rows = pick(1, 1, 2, 3)
        heads = [pick(1, 2, 3) for _ in range(2)]
        ld = [hd + 8 * pick(0, 0, 1, hd // 8, hd // 4, hd // 8 + 3) for _ in range(2)]
        if pick(True, False):
            ld[1] = ld[0]
        span = [(h - 1) * d + hd for h, d in zip(heads, ld)]
        pitch = max(span) + 8 * pick(0, 0, 1, hd // 8, 100)
        apart = pick(-1, 1) * (pitch * pick(0, 0, 0, 1, 2, 3) + 8 * pick(0, 1, hd // 8 - 1, hd // 8, hd // 8 + 1, hd // 4, 3 * hd // 8))
        places = [[base + r * pitch + h * d for r in range(rows) for h in range(n)]
                  for base, n, d in zip((0, apart), heads, ld)]
        common = any(abs(a - b) < hd for a in places[0] for b in places[1])
        q, k = ({"in": base, "out": base, "in_row_ld": pitch, "out_row_ld": pitch, "in_head_ld": d, "out_head_ld": d}
                for base, d in zip((1 << 40, (1 << 40) + 2 * apart), ld))
        a = L.RotaryArgs(rows=rows, q_heads=heads[0], k_heads=heads[1], head_dim=hd, rotary_dim=hd, axes=1, q=L.RotaryRows(**q),
                         k=L.RotaryRows(**k), positions=1 << 20, pos_ld=rows, table=1 << 20)
        assert L.load().t2w_rotary(ctypes.byref(a), None) == (INVALID if common else UNSUPPORTED), (rows, heads, ld, pitch, apart)
        seen[common] += 1
    assert min(seen.values()) > 500


def test_no_turns_are_no_work():
    for kw in (dict(rows=0), dict(q_heads=0, k_heads=0)):
        assert L.load().t2w_rotary(ctypes.byref(rotary_args(**kw)), None) == 0


# ---- quantising -------------------------------------------------------------------------------------------------------


def nearest_even(q):
    f = math.floor(q)
    r = q - f
    return f + (1 if r > 0.5 or (r == 0.5 and f % 2) else 0)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 128])
def test_quantize(dtype, zeros, group):
    gen = torch.Generator().manual_seed(group)
    w = (torch.randn(6, 256, generator=gen) * torch.exp2(torch.randint(-3, 4, (6, 1), generator=gen).float())).to(dtype)
    w[2] = 0
    w[3] = w[3].abs()  # a range that ends at 0
    w[4, 0] = 40.0  # one value far above the others
    codes, scales, z = w4.quantize(w, group, zeros)
    assert codes.dtype == torch.uint8 and scales.dtype == dtype and (z is None) == (not zeros) and int(codes.max()) <= 15
    for r in range(6):
        for g in range(256 // group):
            v = w[r, g * group:(g + 1) * group].double().tolist()
            if zeros:
                low, high = min(0.0, *v), max(0.0, *v)
                s = torch.tensor((high - low) / 15, dtype=torch.float64).to(dtype)
            else:
                s = torch.tensor(max(abs(x) for x in v) / 7, dtype=torch.float64).to(dtype)
            assert torch.equal(scales[r, g], s)
            s = float(s)
            zero = 8 if not zeros else int(z[r, g])
            if zeros:
                assert zero == (0 if s == 0 else min(15, max(0, nearest_even(-low / s))))
            want = [min(15, max(0, (0 if s == 0 else nearest_even(x / s)) + zero)) for x in v]
            assert codes[r, g * group:(g + 1) * group].tolist() == want


@pytest.mark.parametrize("zeros", [False, True])
def test_a_parameter_is_quantised_without_a_gradient(zeros):
    w = torch.randn(6, 128, generator=torch.Generator().manual_seed(1)).to(BF16)
    got, want = w4.quantize(torch.nn.Parameter(w), 64, zeros), w4.quantize(w, 64, zeros)
    for a, b in zip(got, want):
        assert (a is None and b is None) or (torch.equal(a, b) and not a.requires_grad and a.grad_fn is None)


def test_matrices_that_cannot_be_quantised():
    w = torch.randn(4, 128).to(BF16)
    for bad, kw in ((w.float(), {}), (w[0], {}), (w, dict(group=16)), (w[:, :96], dict(group=64)), (w[:, :0], {})):
        with pytest.raises(ValueError):
            w4.quantize(bad, **kw)
    for v in (float("nan"), float("inf")):
        x = w.clone()
        x[1, 2] = v
        with pytest.raises(ValueError):
            w4.quantize(x)


def test_packing_needs_a_gpu():
    codes, scales = torch.zeros(8, 128, dtype=torch.uint8), torch.ones(8, 1, dtype=BF16)
    with pytest.raises(RuntimeError):
        w4.pack(codes, scales)
    with pytest.raises(ValueError):
        w4.pack(codes, scales[:, :0])


# ---- the rotary table -------------------------------------------------------------------------------------------------


def test_table():
    t = Rotary(128, [16, 24, 24], base=1000000.0, device="cpu").table
    assert t.shape == (128,) and t[64:].tolist() == [0] * 16 + [1] * 24 + [2] * 24
    with decimal.localcontext() as c:
        c.prec = 60
        pi = decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494")
        for i in range(64):
            f = decimal.Decimal(1000000) ** (decimal.Decimal(-2 * i) / 128) / (2 * pi) * 2 ** 64
            assert abs(int(t[i]) % 2 ** 64 - f) <= decimal.Decimal("0.5000001")
    assert Rotary(64, [14, 9, 9], interleaved=True, device="cpu").table[32:].tolist() == [0, 1, 2] * 9 + [0] * 5
    own = Rotary(16, inv_freq=[0.0, -1.0, 7.0, 0.5, 1e-9, 2.0, 3.0, 4.0], device="cpu").table
    assert int(own[0]) == 0 and int(own[1]) == -int(Rotary(16, inv_freq=[1.0] * 8, device="cpu").table[0])


@pytest.mark.parametrize("args,kw", [
    ((60,), {}), ((0,), {}), ((64, [16, 15]), {}), ((64, [33, -1]), {}), ((64, []), {}), ((64,), dict(rotary_dim=24)),
    ((64,), dict(rotary_dim=128)), ((64,), dict(pairs="both")), ((64,), dict(base=0.0)), ((64,), dict(base=float("inf"))),
    ((64,), dict(base=float("nan"))), ((64,), dict(inv_freq=[1.0])), ((64,), dict(inv_freq=[float("nan")] * 32))])
def test_tables_that_there_are_not(args, kw):
    with pytest.raises(ValueError):
        Rotary(*args, device="cpu", **kw)
