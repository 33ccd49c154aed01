"""A paged K/V cache held in 8 bits: the step's tables built on the GPU (``plan``), new keys and values quantised into
their pages (``append``), attention over the pages (``attend``), and ``B200PagedCache``, which keeps the buffers of one.

The cache of one layer is a pair of code tensors ``float8_e4m3fn [pages, kv_heads, page, head_dim]`` and a pair of scale
tensors ``fp32 [pages, kv_heads]`` holding powers of two; a value is code * scale.  ``table`` (``int32 [requests,
blocks]``) names the page of each ``page`` tokens of a request and, like the plan, is shared by all layers of a step.

Everything runs on the current stream of the tensors' GPU, reads lengths on the GPU only and never waits for it, so a
step may be captured in a CUDA graph; tensors that were made on another stream are the caller's to order, as with any
torch operator.  What only the GPU can find wrong (pages used up, lengths that do not fit, a free stack that names no page)
makes the plan void: its calls then write zeros for their rows and leave the cache as it was, and ``PagedPlan.check``
raises ``T2WError``.  A call that meets a page which its own codes do not have makes the plan void from itself on.

Arguments that cannot be right raise at the call: ``T2WError`` for sizes that the kernels do not have (page 16, 32, 64 or
128; head_dim 64 or 128; at most 128 query heads to a key head), ``RuntimeError`` for tensors of the wrong type, shape,
device or alignment.
"""

from __future__ import annotations

import torch

from . import lib as L
from . import ops as O


class PagedPlan:
    """One step's tables (see ``plan``): what the kernels read (``buffer``), and views of it,

    ``q_start`` int32 [requests + 1]: the first row of each request, and the rows in use;
    ``kv_len`` int32 [requests]: tokens of each request, this step's among them where they are appended;
    ``slot`` int32 [rows]: page * page_size + place in the page of each row; -1 for padding and for rows not appended;
    ``request`` int32 [rows]: the request of each row; -1 for padding;
    ``free_left`` int32 [1]: the free pages left (where the rows are appended)."""

    __slots__ = ("buffer", "q_start", "kv_len", "slot", "request", "free_left", "table", "requests", "rows", "max_fresh",
                 "page", "q_heads", "kv_heads", "head_dim", "causal")

    def check(self) -> None:
        """Wait for the GPU and raise ``T2WError`` if the plan is void or a call that took it met a fault."""
        L.check("t2w_paged_plan", O.load().paged_status(self.buffer))


def plan(fresh: torch.Tensor, length: torch.Tensor, table: torch.Tensor, page: int, *, rows: int, q_heads: int,
         kv_heads: int, head_dim: int, causal: bool = True, max_fresh: int | None = None,
         free: torch.Tensor | None = None, free_count: torch.Tensor | None = None, kv_len: torch.Tensor | None = None,
         free_left: torch.Tensor | None = None) -> PagedPlan:
    """The tables of a step in which request r brings ``fresh[r]`` rows (0 .. ``max_fresh``, by default ``rows``) to
    ``length[r]`` cached tokens (int32 tensors on the GPU).  The rows of all requests lie one after the other in the
    step's ``rows`` rows; what is left over is padding.

    With ``free`` (int32 [pages], a stack of page numbers) and ``free_count`` (int32 [1]) the rows are to be appended: pages
    are taken off the end of the stack and entered in ``table`` in place.  ``plan.kv_len`` and ``plan.free_left`` are the
    new lengths and the pages left.  ``kv_len`` / ``free_left`` name where to write them too; they may be ``length`` and
    ``free_count`` themselves, which are otherwise left as they are, so that the call can be made again.
    Without ``free`` the rows only look at the ``length[r]`` tokens that are cached.

    ``q_heads``, ``kv_heads``, ``head_dim`` and ``causal`` are those of the attention that will take the plan, whose work it
    splits over the GPU.  A tight ``max_fresh`` matters: at 16 rows to a key head and request or fewer (max_fresh * q_heads /
    kv_heads) the attention runs its form for single tokens."""
    most = rows if max_fresh is None else max_fresh
    p = PagedPlan()
    p.buffer, p.q_start, p.kv_len, p.slot, p.request, p.free_left = O.call(
        "paged_plan", fresh, length, table, page, rows, max(1, most), q_heads, kv_heads, head_dim, causal, free,
        free_count, kv_len, free_left)
    p.table, p.requests, p.rows, p.max_fresh = table, fresh.numel(), rows, max(1, most)
    p.page, p.q_heads, p.kv_heads, p.head_dim, p.causal = page, q_heads, kv_heads, head_dim, causal
    return p


def _fits(p: PagedPlan, codes: torch.Tensor, rows: torch.Tensor, heads: int) -> None:
    if codes.shape[1:] != (p.kv_heads, p.page, p.head_dim):
        raise ValueError(f"the plan is for pages [{p.kv_heads}, {p.page}, {p.head_dim}], the codes are {tuple(codes.shape)}")
    if rows.shape != (p.rows, heads, p.head_dim):
        raise ValueError(f"the plan is for rows [{p.rows}, {heads}, {p.head_dim}], got {tuple(rows.shape)}")


def append(k: torch.Tensor, v: torch.Tensor, k_codes: torch.Tensor, v_codes: torch.Tensor, k_scale: torch.Tensor,
           v_scale: torch.Tensor, plan: PagedPlan) -> None:
    """Round the step's new keys and values ``[rows, kv_heads, head_dim]`` (bf16 or fp16; views with strides of whole
    16-byte pieces, such as columns of fused projection rows) into their pages, in place.

    The scale of a page and head is the least power of two with which the largest magnitude ever given to it fits e4m3
    (at most 448 * 2^64, at least 2^-64).  Where a step's rows raise it, the codes already there are rounded again.  A
    page and head that is given an infinity or a NaN reads as NaN from then on.  Rows whose page these codes do not have
    (fewer pages than the free stack) are not written, and ``PagedPlan.check`` raises."""
    _fits(plan, k_codes, k, plan.kv_heads)
    O.call("paged_append", k, v, k_codes, v_codes, k_scale, v_scale, plan.buffer, plan.requests, plan.max_fresh, plan.q_heads)


def attend(q: torch.Tensor, k_codes: torch.Tensor, v_codes: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
           plan: PagedPlan, scale: float | None = None, lse: bool = False):
    """softmax(scale q k^T) v of the plan's rows ``q [rows, q_heads, head_dim]`` (bf16 or fp16) over their requests' pages;
    ``scale`` is 1 / sqrt(head_dim) unless given.  Returns the output (q's type) and, with ``lse``, the natural log of each
    row's sum of exponentials (fp32 ``[rows, q_heads]``).  A row that sees no key, and padding, gives zeros and -inf."""
    _fits(plan, k_codes, q, plan.q_heads)
    r = O.call("paged_attn", q, k_codes, v_codes, k_scale, v_scale, plan.table, plan.buffer, plan.requests, plan.max_fresh,
               plan.causal, plan.head_dim ** -0.5 if scale is None else scale, lse)
    return tuple(r) if lse else r[0]


def release(done: torch.Tensor, length: torch.Tensor, table: torch.Tensor, page: int, free: torch.Tensor,
            free_count: torch.Tensor, status: torch.Tensor) -> None:
    """Give the pages of the requests with ``done[r] != 0`` back to the free stack; their lengths become 0.  ``status``
    (int32 [1]) becomes T2W_ERR_INVALID, and nothing is given back, where more pages would come back than there are or a
    request's length or table names none."""
    O.call("paged_release", done, length, table, page, free, free_count, status)


class B200PagedCache:
    """The paged cache of ``layers`` attention layers for up to ``requests`` requests of ``max_tokens`` tokens each, in a
    pool of ``pages`` pages that they share.

    A step: ``p = cache.plan(fresh, rows=...)``, then for each layer ``cache.append(layer, k, v, p)`` and
    ``cache.attend(layer, q, p)``.  ``plan`` advances ``cache.length`` and ``cache.free_count`` on the GPU.  A finished
    request's place is given back with ``release``."""

    def __init__(self, layers: int, pages: int, page: int, kv_heads: int, head_dim: int, requests: int, max_tokens: int,
                 q_heads: int | None = None, device="cuda"):
        if min(layers, pages, requests, max_tokens) <= 0:
            raise ValueError("layers, pages, requests and max_tokens are positive")
        self.page, self.kv_heads, self.head_dim, self.q_heads = page, kv_heads, head_dim, q_heads or kv_heads
        n = L.load().t2w_paged_plan_ints(requests, 1, 1, page, self.q_heads, kv_heads, head_dim, None)
        if n < 0:
            raise L.T2WError("t2w_paged_plan_ints", n)
        code = dict(device=device, dtype=torch.float8_e4m3fn)
        self.k = torch.zeros(layers, pages, kv_heads, page, head_dim, **code)
        self.v = torch.zeros(layers, pages, kv_heads, page, head_dim, **code)
        self.k_scale = torch.ones(layers, pages, kv_heads, device=device)
        self.v_scale = torch.ones(layers, pages, kv_heads, device=device)
        self.table = torch.full((requests, -(-max_tokens // page)), -1, device=device, dtype=torch.int32)
        self.length = torch.zeros(requests, device=device, dtype=torch.int32)
        self.free = torch.arange(pages - 1, -1, -1, device=device, dtype=torch.int32)
        self.free_count = torch.full((1,), pages, device=device, dtype=torch.int32)
        self.status = torch.zeros(1, device=device, dtype=torch.int32)

    def plan(self, fresh: torch.Tensor, rows: int, max_fresh: int | None = None, causal: bool = True) -> PagedPlan:
        """The tables of a step that appends ``fresh[r]`` rows to request r, and the caches' new lengths."""
        return plan(fresh, self.length, self.table, self.page, rows=rows, q_heads=self.q_heads, kv_heads=self.kv_heads,
                    head_dim=self.head_dim, causal=causal, max_fresh=max_fresh, free=self.free, free_count=self.free_count,
                    kv_len=self.length, free_left=self.free_count)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, p: PagedPlan) -> None:
        append(k, v, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer], p)

    def attend(self, layer: int, q: torch.Tensor, p: PagedPlan, scale: float | None = None, lse: bool = False):
        return attend(q, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer], p, scale, lse)

    def release(self, done: torch.Tensor) -> None:
        """Give back the pages of the requests with ``done[r] != 0`` (int32 [requests])."""
        release(done, self.length, self.table, self.page, self.free, self.free_count, self.status)

    def check(self) -> None:
        """Wait for the GPU and raise ``T2WError`` if a release went wrong."""
        status = int(self.status)
        self.status.zero_()
        L.check("t2w_paged_release", status)

    def bytes_per_token(self) -> int:
        """Bytes of codes that a token takes over all layers (the scales add 8 bytes for each page, head and layer)."""
        return 2 * self.k.shape[0] * self.kv_heads * self.head_dim
