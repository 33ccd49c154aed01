"""GPU: the paged 8-bit K/V cache where its tables, pools and sizes are at their limits (see ``test_gpu_paged``, whose
64-bit statement and bounds these tests use)."""

import math

import pytest
import torch

from b200t2w import lib as L
from b200t2w import paged
from tests.test_gpu_paged import Model, i32, normal

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _dev():
    assert torch.cuda.is_available()
    assert L.load().t2w_device_ok(torch.cuda.current_device()) == 1


# ---- pools and tables that do not fit -------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_append_to_fewer_pages_than_the_free_stack(dtype):
    """A layer's codes are a view of the first 3 pages of a pool, the free stack has 6: pages 3 to 5 are not written, the
    other rows are, and the status tells."""
    page, heads, hd, have, pages = 16, 2, 64, 3, 6
    pool = [torch.full((pages, heads, page, hd), 0x35, device="cuda", dtype=torch.uint8) for _ in range(2)]
    scales = [torch.full((pages, heads), 3.0, device="cuda") for _ in range(2)]
    codes = [t[:have].view(torch.float8_e4m3fn) for t in pool]
    fresh = [40, 33]  # pages 0, 1, 2 and 3, 4, 5
    m = Model(pages, heads, page, hd, 2, 3)
    table, free, count = torch.full((2, 3), -1, device="cuda", dtype=torch.int32), i32(m.free), i32([pages])
    p = paged.plan(i32(fresh), i32([0, 0]), table, page, rows=73, q_heads=heads, kv_heads=heads, head_dim=hd, max_fresh=40,
                   free=free, free_count=count)
    p.check()
    slots, owner, _ = m.plan(fresh)
    assert p.slot.tolist() == slots
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = [normal(gen, 73, heads, hd, dtype=dtype) for _ in range(2)]
    paged.append(x[0], x[1], codes[0], codes[1], scales[0][:have], scales[1][:have], p)
    with pytest.raises(L.T2WError) as e:
        p.check()
    assert e.value.status == -1
    for w in (0, 1):
        m.append(w, x[w].double().cpu(), slots, owner)
        assert bool((pool[w][have:] == 0x35).all()) and bool((scales[w][have:] == 3.0).all())
        got, scale = codes[w].double().cpu(), scales[w].double().cpu()
        for g in range(have):
            n = min(page, 40 - g * page)  # request 0's
            assert torch.equal(got[g, :, :n], m.codes[w][g, :, :n]) and torch.equal(scale[g], m.scale[w][g])
