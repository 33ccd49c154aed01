"""Timing cases of the paged 8-bit K/V cache: ``paged.plan`` (block tables and slot maps from request lengths),
``paged.append`` (new keys and values quantised into their pages) and ``paged.attend`` (attention over the pages).

Cache of one layer: codes e4m3 ``[pages, kv_heads, page, head_dim]`` for K and for V, and one fp32 scale, a power of two,
for each page and head (``[pages, kv_heads]``).  A value is code * scale.  ``table[r, b]`` is the page that holds tokens
``b * page .. (b + 1) * page - 1`` of request r.

``run`` is one pass through one of the three operators: in elementary torch operations, or with ``own`` through the
package's entry points.
"""

import math
import os
import random
import sys

import torch

own = False

E_MIN, E_MAX = -64, 64  # exponents of the scales
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _paged():
    pkg = os.path.join(os.getcwd(), "minicpm-o-4.5-single-gpu-engine_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from b200t2w import paged

    return paged


# ---- cases ----------------------------------------------------------------------------------------------------------
# fresh: new tokens of each request in this step; length: tokens that each request has in the cache before them (plan,
# append), or all the tokens it has (attend).  Both are spread evenly over [lo, hi] request by request.


def listed():
    return [
        # speech-token decode of 64 streams, one token each: the step's tables before its layers run
        dict(name="plan decode 64x1", op="plan", requests=64, fresh_lo=1, fresh_hi=1, len_lo=17, len_hi=2100, page=16,
             q_heads=32, kv_heads=8, head_dim=128, causal=True),
        # a flow solve's steady windows: both guidance rows of 64 streams, 50 frames each, behind a 300-frame prompt
        dict(name="plan windows 128x50", op="plan", requests=128, fresh_lo=50, fresh_hi=50, len_lo=300, len_hi=400,
             page=64, q_heads=8, kv_heads=8, head_dim=64, causal=False),
        # prompts of many requests admitted at once
        dict(name="plan prompts 256x2k", op="plan", requests=256, fresh_lo=1, fresh_hi=4095, len_lo=0, len_hi=9000,
             page=32, q_heads=16, kv_heads=4, head_dim=128, causal=True),
        # the smallest append: a few streams, one token each, into partly filled pages
        dict(name="append decode 4x1", op="append", requests=4, fresh_lo=1, fresh_hi=1, len_lo=5, len_hi=700, page=16,
             kv_heads=8, head_dim=64, dtype="bf16"),
        # one token of each of 160 requests, wide heads, in half precision
        dict(name="append decode 160x1", op="append", requests=160, fresh_lo=1, fresh_hi=1, len_lo=0, len_hi=1500,
             page=32, kv_heads=8, head_dim=128, dtype="fp16"),
        # steady windows, keys and values taken from the fused q | k | v rows
        dict(name="append windows 128x50", op="append", requests=128, fresh_lo=50, fresh_hi=50, len_lo=300, len_hi=400,
             page=64, kv_heads=8, head_dim=64, dtype="bf16"),
        # ragged prompts, about 65 thousand tokens
        dict(name="append prompts 16x4k", op="append", requests=16, fresh_lo=1900, fresh_hi=6300, len_lo=0, len_hi=333,
             page=64, kv_heads=8, head_dim=128, dtype="bf16"),
        # one stream's single token: latency
        dict(name="attend decode 1x233", op="attend", requests=1, fresh_lo=1, fresh_hi=1, len_lo=233, len_hi=233, page=16,
             q_heads=8, kv_heads=8, head_dim=64, causal=True, dtype="bf16"),
        # 64 streams' single tokens over ragged histories, four query heads to a key head
        dict(name="attend decode 64x4k", op="attend", requests=64, fresh_lo=1, fresh_hi=1, len_lo=40, len_hi=4100,
             page=32, q_heads=32, kv_heads=8, head_dim=128, causal=True, dtype="bf16"),
        # few requests with very long histories (one table row of thousands of pages), half precision
        dict(name="attend decode 3x150k", op="attend", requests=3, fresh_lo=1, fresh_hi=1, len_lo=90001, len_hi=150001,
             page=64, q_heads=16, kv_heads=2, head_dim=128, causal=True, dtype="fp16"),
        # the flow solve's steady windows: every frame sees the cached frames and the whole window
        dict(name="attend windows 128x50", op="attend", requests=128, fresh_lo=50, fresh_hi=50, len_lo=350, len_hi=450,
             page=64, q_heads=8, kv_heads=8, head_dim=64, causal=False, dtype="bf16"),
        # prompts in chunks behind cached tokens, causal, four query heads to a key head
        dict(name="attend chunks 4x1k", op="attend", requests=4, fresh_lo=700, fresh_hi=1024, len_lo=1024, len_hi=4096,
             page=16, q_heads=16, kv_heads=4, head_dim=128, causal=True, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend"])
    page = rng.choice([16, 32, 64, 128])
    hd = rng.choice([64, 128])
    kv = rng.choice([1, 2, 4, 8, 8])
    q_heads = kv * rng.choice([1, 2, 4, 8])
    kind = rng.choice(["decode", "window", "chunk"])
    causal = rng.random() < (0.5 if kind == "window" else 0.9)
    hi = {"decode": 1, "window": _log(rng, 2, 150), "chunk": _log(rng, 150, 1024)}[kind]
    lo = hi if rng.random() < 0.3 else max(1, hi // rng.choice([2, 5]))
    if op == "plan":
        return dict(op=op, requests=_log(rng, 1, 256), fresh_lo=lo, fresh_hi=hi, len_lo=0, len_hi=_log(rng, 1, 9000),
                    page=page, q_heads=q_heads, kv_heads=kv, head_dim=hd, causal=causal)
    if op == "append":
        n = _log(rng, 1, max(1, min(256, 32000 // hi)))
        return dict(op=op, requests=n, fresh_lo=lo, fresh_hi=hi, len_lo=0, len_hi=_log(rng, 1, 1500), page=page,
                    kv_heads=kv, head_dim=hd, dtype=rng.choice(["bf16", "bf16", "fp16"]))
    top = {"decode": 60000, "window": 3000, "chunk": 4096}[kind]
    len_hi = max(hi, _log(rng, max(20, hi), top))
    # no more cached values, and no more query-key pairs, than the largest cases listed
    n = min(128, 60_000_000 // (len_hi * kv * hd), 40_000_000 // (len_hi * hi * q_heads))
    return dict(op=op, requests=_log(rng, 1, max(1, n)), fresh_lo=lo, fresh_hi=hi, len_lo=max(lo, len_hi // 3),
                len_hi=len_hi, page=page, q_heads=q_heads, kv_heads=kv, head_dim=hd, causal=causal,
                dtype=rng.choice(["bf16", "bf16", "fp16"]))


def _lengths(case):
    """Each request's new tokens and cached tokens: by the case alone, so that its work is known without a seed."""
    n = case["requests"]
    r = random.Random("%d %d %d %d %d" % (n, case["fresh_lo"], case["fresh_hi"], case["len_lo"], case["len_hi"]))

    def spread(lo, hi):
        v = [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)] if n > 1 else [hi]
        r.shuffle(v)
        return v

    fresh, length = spread(case["fresh_lo"], case["fresh_hi"]), spread(case["len_lo"], case["len_hi"])
    if case["op"] == "attend":
        length = [max(a, b) for a, b in zip(length, fresh)]
    return fresh, length


# ---- inputs ---------------------------------------------------------------------------------------------------------


def _pow2(amax):
    """The exponent e of the smallest 2^e with amax <= 448 * 2^e, within [E_MIN, E_MAX]."""
    m, e = torch.frexp(amax)
    return torch.where(amax > 0, e - 9 + (m > 0.875).to(e.dtype), torch.full_like(e, E_MIN)).clamp(E_MIN, E_MAX)


def _filled(pages, heads, page, hd, gen):
    """A layer's pages as steps before this one left them: normal keys and values whose size differs by page and head."""
    out = []
    for _ in range(2):
        scale = torch.exp(0.4 * torch.randn(pages, heads, 1, 1, device="cuda", generator=gen))
        codes = torch.empty(pages, heads, page, hd, device="cuda", dtype=torch.float8_e4m3fn)
        scales = torch.empty(pages, heads, device="cuda")
        step = max(1, (1 << 26) // (heads * page * hd))
        for i in range(0, pages, step):
            j = min(pages, i + step)
            x = torch.randn(j - i, heads, page, hd, device="cuda", generator=gen) * scale[i:j]
            s = torch.exp2(_pow2(x.abs().amax((2, 3))).float())
            codes[i:j] = (x / s[:, :, None, None]).to(torch.float8_e4m3fn)
            scales[i:j] = s
        out += [codes, scales]
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    fresh, length = _lengths(case)
    n, page = case["requests"], case["page"]
    grow = case["op"] != "attend"
    held = [-(-x // page) for x in length]  # pages that each request has
    need = [-(-(a + b) // page) if grow else h for a, b, h in zip(length, fresh, held)]
    blocks = max(1, max(need))
    pages = sum(need) + 3
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    table = torch.full((n, blocks), -1, device="cuda", dtype=torch.int32)
    h = torch.tensor(held, device="cuda")
    mine = torch.arange(blocks, device="cuda")[None, :] < h[:, None]
    table[mine] = order[:sum(held)]
    free = torch.cat([order[sum(held):], order[:sum(held)]]).contiguous()
    st = dict(case=case, rows=sum(fresh), max_fresh=max(fresh), table=table, free=free,
              free_count=torch.tensor([pages - sum(held)], device="cuda", dtype=torch.int32),
              fresh=torch.tensor(fresh, device="cuda", dtype=torch.int32),
              length=torch.tensor(length, device="cuda", dtype=torch.int32))
    if case["op"] == "plan":
        return st
    kv, hd, dt = case["kv_heads"], case["head_dim"], TYPES[case["dtype"]]
    st["kc"], st["ks"], st["vc"], st["vs"] = _filled(pages, kv, page, hd, gen)
    if case["op"] == "append":
        # keys and values are columns of the fused projection's rows, as the products before them write them
        qkv = torch.randn(st["rows"], 3, kv, hd, device="cuda", generator=gen)
        qkv *= torch.exp(0.4 * torch.randn(st["rows"], 3, kv, 1, device="cuda", generator=gen))
        qkv = qkv.to(dt)
        st["k"], st["v"] = qkv[:, 1], qkv[:, 2]
        q_heads, causal = kv, True
        st["plain"] = _plan(st)
    else:
        q_heads, causal = case["q_heads"], case["causal"]
        st["q"] = (1.5 * torch.randn(st["rows"], q_heads, hd, device="cuda", generator=gen)).to(dt)
    if own:  # the step's plan, made once and used by each of its layers
        p = _paged()
        more = dict(free=st["free"], free_count=st["free_count"]) if grow else {}
        st["plan"] = p.plan(st["fresh"], st["length"], st["table"], page, rows=st["rows"], max_fresh=st["max_fresh"],
                            q_heads=q_heads, kv_heads=kv, head_dim=hd, causal=causal, **more)
    return st


# ---- one pass -------------------------------------------------------------------------------------------------------


def run(st):
    op = st["case"]["op"]
    if op == "plan":
        return _run_plan(st)
    if op == "append":
        return _run_append(st)
    return _run_attend(st)


def _plan(st):
    """Query offsets, key counts, the table with its new pages, the free pages left, and each row's slot and request."""
    page, fresh, length, table = st["case"]["page"], st["fresh"].long(), st["length"].long(), st["table"]
    kv_len = length + fresh
    q_start = torch.zeros(fresh.numel() + 1, device=fresh.device, dtype=torch.int64)
    q_start[1:] = torch.cumsum(fresh, 0)
    first, last = (length + page - 1) // page, (kv_len + page - 1) // page
    base = torch.cumsum(last - first, 0) - (last - first)
    block = torch.arange(table.shape[1], device=fresh.device)[None, :]
    new = (block >= first[:, None]) & (block < last[:, None])
    nth = base[:, None] + block - first[:, None]  # the nth page taken off the free list's end
    at = (st["free_count"].long() - 1 - nth).clamp(0, st["free"].numel() - 1)
    table.copy_(torch.where(new, st["free"][at], table))
    row = torch.arange(st["rows"], device=fresh.device)
    request = torch.searchsorted(q_start[1:], row, right=True)
    pos = length[request] + row - q_start[request]
    slot = table[request, pos // page].long() * page + pos % page
    i32 = torch.int32
    return dict(q_start=q_start.to(i32), kv_len=kv_len.to(i32), table=table, slot=slot.to(i32), request=request.to(i32),
                free_left=(st["free_count"].long() - (last - first).sum()).to(i32))


def _run_plan(st):
    if not own:
        return _plan(st)
    c = st["case"]
    p = _paged().plan(st["fresh"], st["length"], st["table"], c["page"], rows=st["rows"], max_fresh=st["max_fresh"],
                      q_heads=c["q_heads"], kv_heads=c["kv_heads"], head_dim=c["head_dim"], causal=c["causal"],
                      free=st["free"], free_count=st["free_count"])
    return dict(q_start=p.q_start, kv_len=p.kv_len, table=st["table"], slot=p.slot, request=p.request,
                free_left=p.free_left)


def _append_plain(x, codes, scales, page, slot, length, fresh, table):
    """New rows x into their pages: a page's scale grows to what its new rows need, its older rows are rounded again to
    the grown scale, and the new rows are rounded to it."""
    x = x.float()
    where, off = slot // page, slot % page
    amax = torch.zeros(codes.shape[0], x.shape[1], device=x.device)
    amax = amax.index_reduce(0, where, x.abs().amax(2), "amax")
    # rows that a page held before this step: only the page that a request's new rows begin in has any
    old = torch.zeros(codes.shape[0], device=x.device, dtype=torch.int64)
    cut = (length % page > 0) & (fresh > 0)
    at = table[torch.arange(length.numel(), device=x.device), (length // page).clamp(max=table.shape[1] - 1)].long()
    old.index_add_(0, torch.where(cut, at, 0), torch.where(cut, length % page, 0))
    touched = torch.zeros(codes.shape[0], device=x.device, dtype=torch.bool)
    touched[where] = True
    need = torch.exp2(_pow2(amax).float())
    grown = torch.where((old > 0)[:, None], torch.maximum(need, scales), need)
    scale = torch.where(touched[:, None], grown, scales)
    mend = touched & (old > 0)
    keep = torch.arange(page, device=x.device)[None, None, :, None] < old[:, None, None, None]
    ratio = torch.where(mend[:, None], scales / scale, 1.0)[:, :, None, None]
    again = (codes.float() * ratio).to(codes.dtype)
    raw = torch.where(keep & mend[:, None, None, None], again.view(torch.uint8), codes.view(torch.uint8))
    codes.view(torch.uint8).copy_(raw)
    q = (x / scale[where][:, :, None]).to(codes.dtype)
    codes.view(torch.uint8)[where, :, off] = q.view(torch.uint8)
    scales.copy_(scale)


def _run_append(st):
    if own:
        _paged().append(st["k"], st["v"], st["kc"], st["vc"], st["ks"], st["vs"], st["plan"])
    else:
        p, page = st["plain"], st["case"]["page"]
        args = page, p["slot"].long(), st["length"].long(), st["fresh"].long(), st["table"]
        _append_plain(st["k"], st["kc"], st["ks"], *args)
        _append_plain(st["v"], st["vc"], st["vs"], *args)
    return dict(k=st["kc"], v=st["vc"], k_scale=st["ks"], v_scale=st["vs"])


def _run_attend(st):
    c = st["case"]
    if own:
        out, lse = _paged().attend(st["q"], st["kc"], st["vc"], st["ks"], st["vs"], st["plan"], lse=True)
        return dict(out=out, lse=lse)
    page, kv, hd, n = c["page"], c["kv_heads"], c["head_dim"], c["requests"]
    group, most = c["q_heads"] // kv, st["max_fresh"]
    fresh, length = st["fresh"].long(), st["length"].long()
    at = st["table"].clamp(min=0).long()

    def gathered(codes, scales):
        x = codes[at].float() * scales[at][:, :, :, None, None]  # [n, blocks, kv, page, hd]
        return x.transpose(1, 2).reshape(n, kv, -1, hd)

    k, v = gathered(st["kc"], st["ks"]), gathered(st["vc"], st["vs"])
    q_start = torch.cumsum(fresh, 0) - fresh
    i = torch.arange(most, device=fresh.device)
    row = (q_start[:, None] + i).clamp(max=st["rows"] - 1)
    q = st["q"].float()[row].view(n, most, kv, group, hd).permute(0, 2, 3, 1, 4).reshape(n, kv, group * most, hd)
    s = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(hd)
    j = torch.arange(s.shape[3], device=fresh.device)
    end = length[:, None] - fresh[:, None] + i + 1 if c["causal"] else length[:, None].expand(n, most)
    end = torch.minimum(end, length[:, None])
    see = (j[None, None, :] < end[:, :, None])[:, None, None]  # [n, 1, 1, most, keys]
    s = s.view(n, kv, group, most, -1).masked_fill(~see, -math.inf)
    top = s.amax(4, keepdim=True)
    e = torch.exp(s - torch.where(top > -math.inf, top, 0.0))
    total = e.sum(4, keepdim=True)
    o = torch.matmul((e / total.clamp(min=1e-30)).view(n, kv, group * most, -1), v)
    o = o.view(n, c["q_heads"], most, hd).transpose(1, 2)
    lse = (top + torch.log(total)).view(n, c["q_heads"], most).transpose(1, 2)
    mine = torch.searchsorted(torch.cumsum(fresh, 0), torch.arange(st["rows"], device=fresh.device), right=True)
    nth = torch.arange(st["rows"], device=fresh.device) - q_start[mine]
    return dict(out=o[mine, nth].to(st["q"].dtype), lse=lse[mine, nth].contiguous())


# ---- what a pass cannot do without ----------------------------------------------------------------------------------


def work(case):
    fresh, length = _lengths(case)
    page, rows = case["page"], sum(fresh)
    if case["op"] == "plan":
        new = sum(-(-(a + b) // page) - -(-a // page) for a, b in zip(length, fresh))
        # lengths in; offsets, key counts and the rows' slots and requests out; each new page off the list into the table
        return {"bytes": 4 * (4 * case["requests"] + 2 * rows + 2 * new), "flops": 0}
    kv, hd = case["kv_heads"], case["head_dim"]
    if case["op"] == "append":
        old = sum((a % page) for a, b in zip(length, fresh) if b)
        runs = sum(-(-(a + b) // page) - a // page for a, b in zip(length, fresh) if b)
        # rows in, codes out; what the partly filled pages hold is read; a scale for each page and head that is touched
        return {"bytes": 2 * kv * (rows * hd * 3 + old * hd + 4 * runs), "flops": 2 * 3 * rows * kv * hd}
    q_heads = case["q_heads"]
    pairs = 0
    for f, n in zip(fresh, length):
        pairs += f * n - (f * (f - 1) // 2 if case["causal"] else 0)
    pages = sum(-(-n // page) for n in length)
    return {"bytes": 2 * sum(length) * kv * hd + 2 * 2 * rows * q_heads * hd + 4 * rows * q_heads + pages * (8 * kv + 4),
            "flops": 4 * pairs * q_heads * hd}


# ---- 64 bits --------------------------------------------------------------------------------------------------------


def _round_e4m3(x):
    """To the nearest e4m3 number, ties to the even one: steps of 2^(e - 3) in [2^e, 2^(e + 1)), 2^-9 below 2^-6."""
    _, e = torch.frexp(x)
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return torch.round(x / step) * step


def _exact_append(x, codes, scales, page, length, fresh, table):
    codes, scales, x = codes.double(), scales.double(), x.double()
    row = 0
    for r, (have, more) in enumerate(zip(length, fresh)):
        done = 0
        while done < more:
            b, o = divmod(have + done, page)
            m = min(page - o, more - done)
            g = int(table[r][b])
            new = x[row + done:row + done + m].transpose(0, 1)  # [heads, m, hd]
            amax = new.abs().amax((1, 2))
            e = torch.ceil(torch.log2(amax / 448.0)).clamp(E_MIN, E_MAX)
            # log2 may land on the wrong side of a whole number: 2^e is the least power of two that is enough
            e = torch.where(448.0 * torch.exp2(e) < amax, e + 1, e)
            e = torch.where(448.0 * torch.exp2(e - 1) >= amax, e - 1, e).clamp(E_MIN, E_MAX)
            s = torch.exp2(e)
            if o:
                s = torch.maximum(s, scales[g])
                codes[g, :, :o] = _round_e4m3(codes[g, :, :o] * (scales[g] / s)[:, None, None])
            scales[g] = s
            codes[g, :, o:o + m] = _round_e4m3(new / s[:, None, None])
            done += m
        row += more
    return codes, scales


def exact(case, seed):
    if case["op"] == "plan":
        return None
    st = prepare(case, seed)
    fresh, length = _lengths(case)
    page = case["page"]
    if case["op"] == "append":
        table = st["plain"]["table"].tolist()
        k, ks = _exact_append(st["k"], st["kc"], st["ks"], page, length, fresh, table)
        v, vs = _exact_append(st["v"], st["vc"], st["vs"], page, length, fresh, table)
        return dict(k=k, v=v, k_scale=ks, v_scale=vs)
    kv, hd, q_heads = case["kv_heads"], case["head_dim"], case["q_heads"]
    group = q_heads // kv
    out = torch.zeros(st["rows"], q_heads, hd, device="cuda", dtype=torch.float64)
    lse = torch.full((st["rows"], q_heads), -math.inf, device="cuda", dtype=torch.float64)
    row = 0
    for r, (f, n) in enumerate(zip(fresh, length)):
        at = st["table"][r, :-(-n // page)].long()
        for h in range(kv):
            k = (st["kc"][at, h].double() * st["ks"][at, h].double()[:, None, None]).reshape(-1, hd)[:n]
            v = (st["vc"][at, h].double() * st["vs"][at, h].double()[:, None, None]).reshape(-1, hd)[:n]
            for g in range(h * group, (h + 1) * group):
                s = st["q"][row:row + f, g].double() @ k.T / math.sqrt(hd)
                if case["causal"]:
                    s += torch.full((f, n), -math.inf, device="cuda", dtype=torch.float64).triu(n - f + 1)
                lse[row:row + f, g] = torch.logsumexp(s, 1)
                out[row:row + f, g] = torch.softmax(s, 1) @ v
        row += f
    return dict(out=out, lse=lse)
