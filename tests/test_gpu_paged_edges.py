"""GPU: the paged 8-bit K/V cache where its tables, pools and sizes are at their limits (see ``test_gpu_paged``, whose
64-bit statement and bounds these tests use).

Where values hold codes that are exactly 0, a row's bound needs the weights' smallest step too.  A weight is a half in units
of 2^M, and M is at least 9 below the largest x_j + log2 s_j (s_j: the value scale of key j's page).  Half of a half's
smallest step is 2^-25, so a weight may be off by 2^-34 max_j 2^(x_j + log2 s_j), and an output column d by

    F = 2^-34 max_j (p_j s_j) sum_j |c_jd|      (p: softmax, c: codes)

beside what ``test_gpu_paged`` allows, whose terms go by sum_j p_j |v_jd| alone."""

import ctypes
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


@pytest.mark.parametrize("group,fresh,hd", [(1, 1, 64), (4, 4, 128), (1, 40, 64), (2, 30, 64), (1, 40, 128), (2, 70, 64)])
@pytest.mark.parametrize("entry", [-1, -2, -3, 10, 2 ** 31 - 1, -2 ** 31])
def test_no_entry_outside_the_pool_passes(group, fresh, hd, entry):
    """Whatever an entry outside the pool's 10 pages is, and whichever form reads it, the status tells."""
    c = paged.B200PagedCache(1, 10, 16, 1, hd, 1, 160, q_heads=group)
    x = torch.ones(80, 1, hd, device="cuda", dtype=torch.bfloat16)
    c.append(0, x, x, c.plan(i32([80]), 80, 80))
    p = paged.plan(i32([fresh]), c.length, c.table, 16, rows=fresh, q_heads=group, kv_heads=1, head_dim=hd, max_fresh=fresh,
                   causal=False)
    q = torch.ones(fresh, group, hd, device="cuda", dtype=torch.bfloat16)
    c.attend(0, q, p)
    p.check()
    for block in (0, 1, 4):
        kept = c.table[0, block].clone()
        c.table[0, block] = entry
        c.attend(0, q, p)
        with pytest.raises(L.T2WError) as e:
            p.check()
        assert e.value.status == -1
        c.table[0, block] = kept
        p.buffer[4] = 0


@pytest.mark.parametrize("group,fresh,hd", [(1, 1, 64), (4, 3, 128), (2, 30, 64), (1, 40, 128), (4, 100, 64)])
def test_an_entry_outside_the_pool_makes_the_plan_void(group, fresh, hd):
    """Request 1's table names a page that there is not: no row, of no request, is answered from other pages than its own,
    neither in that call nor in the plan's next ones."""
    n, pad = 3, 5
    c = paged.B200PagedCache(1, 60, 16, 2, hd, n, 320, q_heads=2 * group)
    gen = torch.Generator(device="cuda").manual_seed(fresh)
    k = normal(gen, 480, 2, hd)
    c.append(0, k, k, c.plan(i32([200, 120, 160]), 480, 200))
    rows = n * fresh + pad
    p = paged.plan(i32([fresh] * n), c.length, c.table, 16, rows=rows, q_heads=2 * group, kv_heads=2, head_dim=hd,
                   max_fresh=fresh)
    q = normal(gen, rows, 2 * group, hd)
    want = c.attend(0, q, p, lse=True)
    p.check()
    kept = c.table[1, 3].clone()
    c.table[1, 3] = 60
    for entry in (60, kept):  # once void, void for the next layers too
        c.table[1, 3] = entry
        out, lse = c.attend(0, q, p, lse=True)
        with pytest.raises(L.T2WError) as e:
            p.check()
        assert e.value.status == -1
        assert not out.any() and bool((lse == -math.inf).all())
    again = paged.plan(i32([fresh] * n), c.length, c.table, 16, rows=rows, q_heads=2 * group, kv_heads=2, head_dim=hd,
                       max_fresh=fresh)
    got = c.attend(0, q, again, lse=True)
    again.check()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("requests,most,page", [(2, 20, 16), (40, 200, 16), (1100, 5, 32), (1700, 9, 16)])
@pytest.mark.parametrize("where", ["first taken", "last taken", "page begun", "not taken"])
@pytest.mark.parametrize("entry", [-1, 1 << 20, -2 ** 31])
def test_plans_of_lists_that_name_no_page(requests, most, page, where, entry):
    """A free list, or a table's page that rows go into, with an entry that is no page: the plan is void and nothing has
    changed.  An entry that the step does not take does not matter."""
    gen = torch.Generator().manual_seed(requests)
    length = torch.randint(0, 100, (requests,), generator=gen).tolist()
    fresh = torch.randint(0, most + 1, (requests,), generator=gen).tolist()
    length[-1], fresh[-1] = page + 1, most
    blocks = max(-(-(a + b) // page) for a, b in zip(length, fresh))
    pages = sum(-(-(a + b) // page) for a, b in zip(length, fresh)) + 4
    m = Model(pages, 1, page, 1, requests, blocks)
    m.plan(length)
    count, taken = len(m.free), len(m.free) - 4
    free, table = m.free + [0] * (pages - count), [list(t) for t in m.table]
    if where == "first taken":
        free[count - 1] = entry
    elif where == "last taken":
        free[count - taken] = entry
    elif where == "page begun":
        table[-1][1] = entry
    else:
        free[count - taken - 1] = entry
        table[-1][0] = entry
    dev = dict(free=i32(free), table=i32(table), count=i32([count]), length=i32(length), left=i32([count]))
    before = {k: v.clone() for k, v in dev.items()}
    rows = sum(fresh) + 3
    p = paged.plan(i32(fresh), dev["length"], dev["table"], page, rows=rows, q_heads=1, kv_heads=1, head_dim=64, max_fresh=most,
                   free=dev["free"], free_count=dev["count"], kv_len=dev["length"], free_left=dev["left"])
    if where == "not taken":
        p.check()
        assert p.slot.tolist() == m.plan(fresh)[0] + [-1] * 3 and dev["left"].tolist() == [4]
        assert dev["length"].tolist() == m.length
        return
    with pytest.raises(L.T2WError) as e:
        p.check()
    assert e.value.status == -1
    for k, v in dev.items():
        assert torch.equal(v, before[k]), k
    assert p.slot.tolist() == [-1] * rows and p.request.tolist() == [-1] * rows
    assert p.q_start.tolist() == [0] * (requests + 1) and p.kv_len.tolist() == length and p.free_left.tolist() == [count]


@pytest.mark.parametrize("offset", [0, 1, 2, 3])
@pytest.mark.parametrize("pages", [1023, 1025, 1030, 5000])
def test_every_page_taken_is_looked_at(offset, pages):
    """One request takes `pages` pages of a list that lies `offset` entries past a 16-byte boundary: an entry that is no
    page is found wherever it is, and those beside the taken ones are not looked at."""
    held = i32([7] * offset + [-1] + list(range(pages)) + [-1] * 3)
    free, count, one = held[offset:], i32([pages + 1]), i32([pages * 16])
    table = torch.full((1, pages), -1, device="cuda", dtype=torch.int32)

    def plan():
        return paged.plan(one, i32([0]), table, 16, rows=pages * 16, q_heads=1, kv_heads=1, head_dim=64, free=free,
                          free_count=count)

    p = plan()
    p.check()
    assert p.free_left.tolist() == [1] and table[0].tolist() == list(range(pages - 1, -1, -1))
    table.fill_(-1)
    for at in [1, 2, 3, 4, 5, 6, 7, 8, pages // 2, *range(pages - 1030, pages - 1018), pages - 1, pages]:
        if at < 1:
            continue
        free[at] = pages + 4
        with pytest.raises(L.T2WError):
            plan().check()
        assert bool((table == -1).all())
        free[at] = at - 1


def table_of(lens, page, blocks, spare=0):
    """A table that gives each request its pages in order, the free list of the `spare` pages left, and the entries."""
    table, i = [], 0
    for n in lens:
        held = -(-n // page)
        table.append(list(range(i, i + held)) + [-1] * (blocks - held))
        i += held
    return table, list(range(i, i + spare)) + [0] * i, i + spare


@pytest.mark.parametrize("lens", [[150001], [0], [17] * 5 + [0, 3000, 1], [1] * 1024, [33] * 1025,
                                  [r % 70 for r in range(4097)], [r % 70 for r in range(9000)]])
def test_release_of_many_pages(lens):
    """Some requests end, then all of them, some of those without a page; the pages come back in request and block order."""
    page, n = 16, len(lens)
    table, free, pages = table_of(lens, page, -(-max(max(lens), 1) // page) + 1, spare=3)
    dev = dict(length=i32(lens), table=i32(table), free=i32(free), count=i32([3]), status=i32([0]))
    want, free, left = list(lens), free[:3], [list(t) for t in table]
    for done in ([int(r % 3 == n % 3) for r in range(n)], [1] * n):
        paged.release(i32(done), dev["length"], dev["table"], page, dev["free"], dev["count"], dev["status"])
        for r in range(n):
            if done[r]:
                free += [g for g in left[r] if g >= 0]
                want[r], left[r] = 0, [-1] * len(left[r])
        assert dev["status"].tolist() == [0] and dev["count"].tolist() == [len(free)]
        assert dev["free"].tolist()[:len(free)] == free and dev["length"].tolist() == want and dev["table"].tolist() == left
    assert len(free) == pages


@pytest.mark.parametrize("requests", [1, 3, 1024, 1025, 4096, 4097, 9000])
@pytest.mark.parametrize("what", ["length", "negative", "entry", "count", "twice"])
def test_release_that_cannot_be_gives_nothing_back(requests, what):
    """The last request's length or table is wrong, or it alone makes more free pages than there are."""
    page, lens = 16, [20 + r % 60 for r in range(requests)]
    table, free, pages = table_of(lens, page, 6, spare=2)
    if what == "length":
        lens[-1] = 6 * page + 1
    elif what == "negative":
        lens[-1] = -1
    elif what == "entry":
        table[-1][1] = pages
    count = {"count": -1, "twice": 3}.get(what, 2)
    dev = dict(length=i32(lens), table=i32(table), free=i32(free), count=i32([count]), status=i32([0]))
    before = {k: v.clone() for k, v in dev.items()}
    paged.release(i32([1] * requests), dev["length"], dev["table"], page, dev["free"], dev["count"], dev["status"])
    assert dev["status"].tolist() == [-1]
    for k in ("length", "table", "free", "count"):
        assert torch.equal(dev[k], before[k]), k


# ---- many segments and long walks -----------------------------------------------------------------------------------


def on_gpu(k, codes, scale_v, q, scale, causal):
    """``test_gpu_paged.attention`` in 64 bits on the GPU, all rows at once: q [f, hd], k and V's codes [n, hd], V's scales
    [n] -> out, lse, A, B, F."""
    f, n = q.shape[0], k.shape[0]
    s = (q @ k.T) * scale
    b = (q.abs() @ k.abs().T) * scale
    see = torch.ones(f, n, device="cuda", dtype=torch.bool)
    if causal:
        see = torch.arange(n, device="cuda")[None, :] <= torch.arange(n - f, n, device="cuda")[:, None]
    s, b = s.masked_fill(~see, -math.inf), b.masked_fill(~see, 0.0)
    p, v = torch.softmax(s, 1), codes * scale_v[:, None]
    far = 2.0 ** -34 * (p * scale_v).amax(1, keepdim=True) * (see.double() @ codes.abs())
    return p @ v, torch.logsumexp(s, 1), p @ v.abs(), b.amax(1), far


def held(out, lse, ref):
    """Whether out [f, hd] and lse [f], of rows that see a key each, are within the bounds of on_gpu()'s ref."""
    o, l, A, B, far = ref
    u = 2.0 ** -8 if out.dtype == torch.bfloat16 else 2.0 ** -10
    d = (out.double() - o).abs() / (u * o.abs() + (2.0 ** -10 + 2.0 ** -15 * B[:, None]) * A + far + 1e-30)
    assert float(d.max()) <= 1, float(d.max())
    d = (lse.double() - l).abs() / (2.0 ** -16 * B + 2.0 ** -19 * l.abs().clamp(min=1))
    assert float(d.max()) <= 1, float(d.max())


class Filled:
    """A layer's pages filled with codes and scales directly, a request's pages in any order, and attention calls that
    look at them held against 64 bits."""

    def __init__(self, lens, page, heads, hd, seed):
        self.lens, self.page, self.heads, self.hd = lens, page, heads, hd
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        held = [-(-n // page) for n in lens]
        pages = sum(held) + 2
        order = torch.randperm(pages, device="cuda", generator=self.gen).to(torch.int32)
        self.table = torch.full((len(lens), max(1, max(held))), -1, device="cuda", dtype=torch.int32)
        self.at, i = [], 0
        for r, n in enumerate(held):
            self.table[r, :n] = order[i:i + n]
            self.at.append(order[i:i + n].long())
            i += n
        self.codes, self.scales = [], []
        for _ in range(2):
            e = torch.randint(-2, 3, (pages, heads), device="cuda", generator=self.gen)
            self.scales.append(torch.exp2(e.float()))
            self.codes.append(torch.randn(pages, heads, page, hd, device="cuda", generator=self.gen).to(torch.float8_e4m3fn))
        self.length = i32(lens)

    def held_in(self, w, r, h):
        """Codes [n, hd] and scales [n] of request r's keys."""
        at, n = self.at[r], self.lens[r]
        scale = self.scales[w][at, h].double().repeat_interleave(self.page)
        return self.codes[w][at, h].double().reshape(-1, self.hd)[:n], scale[:n]

    def plan(self, fresh, q_heads, causal):
        return paged.plan(i32(fresh), self.length, self.table, self.page, rows=sum(fresh), max_fresh=max(fresh),
                          q_heads=q_heads, kv_heads=self.heads, head_dim=self.hd, causal=causal)

    def attend(self, q, p, **kw):
        return paged.attend(q, self.codes[0], self.codes[1], self.scales[0], self.scales[1], p, **kw)

    def check(self, fresh, group, causal, requests, dtype=torch.bfloat16):
        """One call; the rows of ``requests`` are held against 64 bits, every row against a second call's."""
        heads = self.heads * group
        p = self.plan(fresh, heads, causal)
        q = normal(self.gen, sum(fresh), heads, self.hd, dtype=dtype)
        out, lse = self.attend(q, p, lse=True)
        p.check()
        again, lse2 = self.attend(q, p, lse=True)
        assert torch.equal(out, again) and torch.equal(lse, lse2)
        for r in requests:
            a = sum(fresh[:r])
            if not fresh[r]:
                continue
            if not self.lens[r]:
                assert not out[a:a + fresh[r]].any() and bool((lse[a:a + fresh[r]] == -math.inf).all())
                continue
            for h in range(heads):
                rows = slice(a, a + fresh[r])
                kc, ks = self.held_in(0, r, h // group)
                held(out[rows, h], lse[rows, h], on_gpu(kc * ks[:, None], *self.held_in(1, r, h // group),
                                                        q[rows, h].double(), self.hd ** -0.5, causal))
        return p


def form_of(most, group, hd):
    """Query tokens and keys of a tile, workers of an SM and the tiles that a segment's start counts, by the rows that a
    request has for a key head at most."""
    if most * group <= 16:
        return most, 32, 8 * (1 if hd == 128 or most * group > 8 else 2), 4
    if hd == 64 and most * group <= 64:
        return 64 // group, 64, 4, 2
    return 128 // group, 64, 2, 4


def segments(fresh, lens, heads, causal, tq, kt):
    """(request, key head, query tile, key tiles) of every segment in order."""
    for r, (f, n) in enumerate(zip(fresh, lens)):
        for h in range(heads):
            for q in range(-(-f // tq)):
                sees = max(0, n - max(0, f - (q + 1) * tq)) if causal else n
                yield r, h, q, max(1, -(-sees // kt))


@pytest.mark.parametrize("hd,group,most", [
    (64, 1, 4000), (64, 2, 900), (128, 3, 2000), (128, 5, 700), (128, 7, 900), (64, 8, 300), (128, 16, 700), (64, 100, 50),
    (128, 128, 40), (64, 3, 21), (64, 1, 40), (128, 2, 8)])
@pytest.mark.parametrize("causal", [True, False])
def test_tiles_of_a_plan(hd, group, most, causal):
    """The plan's number of key tiles, for requests that are longer than their rows, shorter, and empty."""
    gen = torch.Generator().manual_seed(group)
    n, heads = 60, 3
    fresh = torch.randint(0, most + 1, (n,), generator=gen).tolist()
    lens = [torch.randint(0, top, (1,), generator=gen).item() for top in (1, 70, most + 1, 3 * most, 20000) for _ in range(12)]
    fresh[5] = most
    table = torch.full((n, -(-max(lens) // 16)), -1, device="cuda", dtype=torch.int32)
    p = paged.plan(i32(fresh), i32(lens), table, 16, rows=sum(fresh), max_fresh=most, q_heads=heads * group, kv_heads=heads,
                   head_dim=hd, causal=causal)
    p.check()
    tq, kt = form_of(most, group, hd)[:2]
    all_of = list(segments(fresh, lens, heads, causal, tq, kt))
    assert int(p.buffer[1]) == sum(s[3] for s in all_of) + int(p.buffer[7]) * len(all_of)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lens,group,heads", [((33, 64), 4, 8), ((17, 60), 5, 8), ((64, 64), 2, 16), ((1, 130), 8, 4)])
def test_many_short_prompts(hd, lens, group, heads):
    """Causal prompts of a tile of keys or two: a worker walks many segments of one tile each, one right after the other."""
    n = 300
    lens = [lens[0] + (7 * r) % (lens[1] - lens[0] + 1) for r in range(n)]
    c = Filled(lens, 16, heads, hd, hd + group)
    p = c.check(lens, group, True, range(0, n, 23))
    workers, segments = int(p.buffer[3]), sum(-(-f // (128 // group)) for f in lens) * heads
    assert segments >= 9 * workers, (segments, workers)


def starts_of(p):
    """A plan's workers' starts: [[request, head, query tile, key tile, first row, rows, keys, place], ..] and the last place."""
    at = (ctypes.c_int64 * 4)()
    assert L.load().t2w_paged_plan_ints(p.requests, p.rows, p.max_fresh, p.page, p.q_heads, p.kv_heads, p.head_dim, at) > 0
    up = lambda n: -(-n // 4) * 4  # noqa: E731
    begin = at[3] + up(p.rows) + 4 * up(p.requests + 1)
    workers = int(p.buffer[3])
    return p.buffer[begin:begin + 8 * (workers + 1)].view(-1, 8).tolist()


def walk(p, fresh, lens, sms):
    """Goes through a plan's split as the workers and the joining do, and checks that every key tile has one worker and that
    of each cut segment the parts are read that were written, once.  Returns how many segments were cut."""
    group = p.q_heads // p.kv_heads
    tq, kt, per_sm, extra_at_most = form_of(p.max_fresh, group, p.head_dim)
    few = p.max_fresh * group <= 16
    tiles, per, workers, extra = int(p.buffer[1]), int(p.buffer[2]), int(p.buffer[3]), int(p.buffer[7])
    assert extra in (0, extra_at_most) and workers <= per_sm * sms
    row0 = [0]
    for n in fresh:
        row0.append(row0[-1] + n)
    segs, place = [], 0
    for r, h, q, nt in segments(fresh, lens, p.kv_heads, p.causal, tq, kt):
        segs.append((r, h, q, nt, place + extra))
        place += nt + extra
    assert place == tiles
    at = {s[:3]: i for i, s in enumerate(segs)}
    starts = starts_of(p)
    places = [s[7] for s in starts]
    assert places[0] == 0 and places[-1] == tiles and all(a <= b for a, b in zip(places, places[1:]))
    if few:
        assert places[:-1] == [w * per for w in range(workers)]
    bw = 8 if few else 1
    written = {}  # by segment: the parts' slots in the order of their keys
    for w in range(workers):
        r, h, q, k, first, rows, keys, begin = starts[w]
        if begin == tiles:  # (moved to the end: nothing is left)
            continue
        i = at[r, h, q]
        assert (first, rows, keys) == (row0[r], fresh[r], lens[r]) and segs[i][4] + k == begin and -extra <= k < segs[i][3]
        j, stop = i, places[w + 1]
        while j < len(segs) and segs[j][4] < stop:
            nt, zero = segs[j][3:]
            lo, hi = max(0, begin - zero), min(nt, stop - zero)
            assert lo < hi
            if hi - lo < nt:
                b = w // bw
                full = bw > 1 and (b + 1) * bw <= workers and zero <= b * bw * per and zero + nt >= (b + 1) * bw * per
                if not full:
                    written.setdefault(j, []).append(2 * w + (j != i))
                elif w % bw == 0:
                    written.setdefault(j, []).append(2 * w)
            j += 1
    joined = {}
    for w in range(1, workers):
        r, h, q, k, first, rows, keys, begin = starts[w]
        zero, before = begin - k, places[w - 1]
        if not (k > 0 and zero >= before):
            continue
        i = at[r, h, q]
        end = zero + segs[i][3]
        w0, last = w - 1, (end - 1) // per
        b0, b1 = -(-zero // (bw * per)), end // (bw * per)
        mid = b1 - b0 if bw > 1 and b1 > b0 else 0
        lead = b0 * bw - w0 if mid else last - w0 + 1
        slots = [2 * (w0 + x) + (x == 0 and zero - extra > before) for x in range(lead)]
        slots += [2 * bw * (b0 + x) for x in range(mid)]
        if mid:
            slots += [2 * x for x in range(b1 * bw, last + 1)]
        assert i not in joined
        joined[i] = slots
    assert joined == written
    return len(joined)


@pytest.mark.parametrize("hd,group,fresh", [(64, 1, 1), (128, 4, 3), (64, 1, 40), (64, 2, 70), (128, 2, 100)])
@pytest.mark.parametrize("zeros", ["first", "last", "every other"])
def test_pages_of_zeros_beside_large_values(hd, group, fresh, zeros):
    """Pages whose values are all 0 have the least scale, 2^-64: beside values of a scale up to 2^26, the other end of what the
    sums of weights hold in full, they still count in the sums."""
    c = Filled([600], 16, 1, hd, fresh)
    for i, g in enumerate(c.at[0].tolist()):
        none = {"first": i < 19, "last": i >= 19, "every other": i % 2 == 0}[zeros]
        c.scales[1][g] = 2.0 ** -64 if none else 2.0 ** 26
        if none:
            c.codes[1].view(torch.uint8)[g] = 0
    c.check([fresh], group, True, [0])


LONG = [
    # head_dim, key heads, query heads to each, most rows, causal, page, requests' keys, dtype
    (64, 8, 1, 1, True, 16, (64, 40, 4000), torch.bfloat16),
    (64, 8, 1, 1, True, 32, (64, 40, 1500, 40000), torch.float16),
    (64, 8, 2, 5, True, 64, (64, 40, 3000), torch.bfloat16),
    (128, 8, 4, 1, True, 32, (64, 40, 3000), torch.float16),
    (128, 4, 8, 2, False, 16, (96, 2, 3000), torch.bfloat16),
    (128, 4, 3, 4, True, 128, (128, 4, 900, 30000), torch.bfloat16),
    (64, 8, 1, 50, False, 64, (128, 50, 700), torch.bfloat16),
    (64, 8, 1, 60, True, 16, (100, 60, 900), torch.float16),
    (64, 5, 3, 20, True, 32, (128, 20, 900, 9000), torch.bfloat16),
    (64, 4, 2, 100, True, 16, (64, 100, 1200), torch.bfloat16),
    (64, 8, 4, 33, False, 128, (100, 33, 300, 9000), torch.float16),
    (128, 4, 4, 60, True, 64, (64, 60, 1200), torch.bfloat16),
    (128, 1, 128, 2, True, 32, (300, 2, 900, 9000), torch.float16),
    (128, 3, 5, 90, False, 16, (64, 90, 500), torch.bfloat16),
]


@pytest.mark.parametrize("hd,heads,group,most,causal,page,keys,dtype", LONG)
def test_calls_with_many_tiles_for_a_worker(hd, heads, group, most, causal, page, keys, dtype):
    """Every form where a worker walks several segments and each segment's start counts places: ragged lengths, requests
    without rows and without keys, here and there one that is far longer than the others."""
    n, lo, hi = keys[:3]
    gen = torch.Generator().manual_seed(hd + group + most)
    lens = [max(most, x) for x in torch.randint(lo, hi + 1, (n,), generator=gen).tolist()]
    fresh = torch.randint(max(1, most // 2), most + 1, (n,), generator=gen).tolist()
    for r in (0, 7, n // 2, n - 1):
        fresh[r] = 0
    for r in (3, 11, n - 2):
        lens[r] = 0
    fresh[5] = most
    lens[9:10] = keys[3:] or lens[9:10]
    c = Filled(lens, page, heads, hd, most)
    p = c.check(fresh, group, causal, [1, 2, 3, 5, 9, n // 2 + 1, n - 2], dtype=dtype)
    assert int(p.buffer[7]) > 0
    assert walk(p, fresh, lens, torch.cuda.get_device_properties(0).multi_processor_count) > 0


@pytest.mark.parametrize("hd,heads,group,most,lens", [
    (64, 2, 1, 1, [5000, 1, 64, 900]), (64, 1, 4, 4, [9000]), (128, 1, 1, 1, [30, 33, 31]), (128, 2, 2, 8, [700, 6011]),
    (64, 2, 2, 30, [900, 64, 65, 3000]), (64, 1, 1, 40, [40]), (64, 2, 2, 70, [900, 4000, 70]), (128, 1, 4, 200, [200, 1000]),
    (128, 2, 3, 300, [300, 5000])])
@pytest.mark.parametrize("causal", [True, False])
def test_calls_with_few_tiles_for_a_worker(hd, heads, group, most, lens, causal):
    """The same walk where starts count nothing."""
    fresh = [max(1, most - r) for r in range(len(lens))]
    lens = [max(a, b) for a, b in zip(lens, fresh)]
    c = Filled(lens, 16, heads, hd, most)
    p = c.check(fresh, group, causal, range(len(lens)))
    assert int(p.buffer[7]) == 0
    walk(p, fresh, lens, torch.cuda.get_device_properties(0).multi_processor_count)
