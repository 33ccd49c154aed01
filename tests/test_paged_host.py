"""CPU: the sizes that the paged cache's C entry points take and refuse.  No GPU work is enqueued here."""

import ctypes

import pytest

from b200t2w import lib as L

INVALID, UNSUPPORTED = -1, -5


def ints(requests=4, rows=64, max_fresh=16, page=16, q_heads=8, kv_heads=2, head_dim=64, status=None):
    return L.load().t2w_paged_plan_ints(requests, rows, max_fresh, page, q_heads, kv_heads, head_dim, status)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("group", [1, 2, 3, 8, 100, 128])
def test_plans_that_there_are(page, head_dim, group):
    n = ints(page=page, head_dim=head_dim, q_heads=2 * group)
    # header, offsets, lengths, a slot and a request for each row, each rounded up to 16 bytes
    assert n >= 8 + 8 + 4 + 64 + 64 and n % 4 == 0
    assert ints(page=page, head_dim=head_dim, q_heads=2 * group, rows=6400) >= n + 2 * (6400 - 64)
    assert ints(page=page, head_dim=head_dim, q_heads=2 * group, rows=0) > 0


@pytest.mark.parametrize("kw,status", [
    (dict(requests=0), INVALID), (dict(rows=-1), INVALID), (dict(max_fresh=0), INVALID), (dict(page=8), INVALID),
    (dict(page=48), INVALID), (dict(page=256), INVALID), (dict(q_heads=3), INVALID), (dict(kv_heads=0), INVALID),
    (dict(head_dim=96), UNSUPPORTED), (dict(head_dim=256), UNSUPPORTED), (dict(q_heads=258), UNSUPPORTED)])
def test_plans_that_there_are_not(kw, status):
    assert ints(**kw) == status


def test_workspace():
    size = L.load().t2w_paged_workspace_bytes
    for head_dim in (64, 128):
        # two parts for each worker, of a row's head_dim sums, its exponent and its sum
        few, many = size(1, 8, 2, head_dim), size(700, 8, 2, head_dim)
        assert few > 0 and few % (2 * 16 * (head_dim + 2) * 4) == 0
        assert many > 0 and many % (2 * 128 * (head_dim + 2) * 4) == 0
    assert size(0, 8, 2, 64) == 0 and size(1, 8, 3, 64) == 0 and size(1, 8, 2, 96) == 0


def test_no_arguments():
    lib = L.load()
    for f in (lib.t2w_paged_plan, lib.t2w_paged_append, lib.t2w_paged_attn):
        assert f(None, None) == INVALID
    for f, t in ((lib.t2w_paged_plan, L.PagedPlanArgs), (lib.t2w_paged_append, L.PagedAppendArgs),
                 (lib.t2w_paged_attn, L.PagedAttnArgs)):
        assert f(ctypes.byref(t()), None) < 0  # all zeros: pointers that are missing
