"""Key/value cache in 4 bits for requests of unequal lengths: pages of 64 slots that a stack of free ones gives out on the GPU, keys and values rounded
by groups of a head's dimensions as they are appended, and softmax attention that reads the codes.

A serving step, per layer after the first two lines:

    cache = PagedCache4(n_layer, n_head, head_size, pages=..., requests=..., max_length=...)
    plan = cache.plan(rows, counts, tokens)            # which slots the step's tokens get: request rows[i] brings counts[i] of the `tokens` rows
    q = cache.append(layer, plan, q, k, v, rope=table) # rows [tokens, heads, head_size]; turns queries and keys where a table is given
    y = cache.attend(layer, plan, q)                   # every token over its request's keys at and before its position
    cache.truncate(rows, lengths)                      # afterwards: drafts that were rejected; length 0 ends a request
    cache.fork(rows, into)                             # requests into[i] become copies of rows[i], sharing their pages (PagedCache4(.., share=True))

Nothing looks at lengths on the host, so that a captured step serves requests of any lengths.  All of it goes to the current stream of the
cache's device: on another stream a step waits for the one before it, and a plan is kept until its kernels there are done.  A group of values x is held as

    lo = min(x),  s = T((max(x) - lo) * (1/15)),  code = min(max(rint((x - lo) / s), 0), 15) in fp32,       standing for code * s + lo

with s and lo in the cache's type T: the smallest value is exact, and the error of the others is half of s at most, and s/15 2^-8 (bf16) or 2^-11 (fp16) of
the group's range more at its upper end, where the rounding of s may leave 15 s short of it.
"""
from __future__ import annotations

import contextlib
import ctypes as C
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _native as N

_NOTHING = contextlib.nullcontext()
_current_device = N._current_device or torch.cuda.current_device

Whole = Union[torch.Tensor, Sequence[int]]

REASONS = {1: "there are not enough free pages", 2: "it would be longer than it may be, or brings more tokens than the plan's max_count",
           3: "there is no such request, or an earlier sequence names it, or its count is negative", 4: "its tokens lie behind the step's rows"}


class CachePlan:
    """A step's place in the cache, as int32 tensors on the GPU: ``starts [B + 1]`` first row of every sequence, ``ends [B]`` tokens held after the step (0:
    refused), ``status [B]`` (0, or why a sequence got nothing: ``REASONS``), ``positions [T]`` and ``slots [T]`` (page * 64 + place in it) of the
    tokens, -1 for those of refused sequences and behind the last one."""

    def __init__(self, cache: "PagedCache4", B: int, T: int, max_count: int):
        self.cache, self.B, self.T, self.max_count, self.step = cache, B, T, max_count, cache._step
        work, self.scratch_bytes = cache._sizes(B, T, max_count)
        self._data, self._first = cache.lengths.new_empty(work + 4 * B + 1 + 2 * T), work
        self._work = N.ptr(self._data)
        self._out = self._work + 4 * work
        self._positions = self._out + 4 * (4 * B + 1)
        self._slots = self._positions + 4 * T

    def _part(self, first: int, n: int) -> torch.Tensor:
        first += self._first
        return self._data[first:first + n]

    @property
    def starts(self) -> torch.Tensor:
        return self._part(0, self.B + 1)

    @property
    def ends(self) -> torch.Tensor:
        return self._part(self.B + 1, self.B)

    @property
    def status(self) -> torch.Tensor:
        return self._part(2 * self.B + 1, self.B)

    @property
    def request(self) -> torch.Tensor:
        return self._part(3 * self.B + 1, self.B)

    @property
    def positions(self) -> torch.Tensor:
        return self._part(4 * self.B + 1, self.T)

    @property
    def slots(self) -> torch.Tensor:
        return self._part(4 * self.B + 1 + self.T, self.T)

    def check(self) -> None:
        """Raise if a sequence was refused.  Waits for the GPU."""
        for i, s in enumerate(self.status.tolist()):
            if s:
                raise RuntimeError(f"sequence {i} of the step was refused: {REASONS[s]}")


class PagedCache4:
    PAGE = 64

    def __init__(self, n_layer: int, n_head: int, head_size: int, *, n_kv_head: Optional[int] = None, pages: int, requests: int, max_length: int,
                 group: int = 64, dtype: torch.dtype = torch.bfloat16, device="cuda", share: bool = False):
        """``pages`` of 64 slots for up to ``requests`` requests of up to ``max_length`` tokens; heads of 32, 64 or 128, codes by ``group``s of 32, 64 or 128
        of their dimensions.  ``n_kv_head`` key/value heads serve ``n_head`` query heads, neighbours the same one.  ``share``: requests may be forked, and steps
        walk pages that neighbouring sequences share once.  Steps whose requests share none are slower than without it (attention 1.1 to 1.75 times, a plan of 8, 64 and 512
        sequences 9, 7 and 11 us -> 14, 21 and 69), and fp16 results over pages that more than 32 queries of a key head share are a little less exact (values of 11 bits meet the
        weights: 0.00027 of the norm off where a walk of one's own is 0.00021; of bf16 both are the rounding of the results)."""
        n_kv_head = n_head if n_kv_head is None else n_kv_head
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError(f"the paged cache lives on CUDA (sm_100a) only, not on {device}")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"a paged cache of {dtype} (torch.bfloat16 or torch.float16)")
        page_bytes = N.call_ret("ll_kv4_page_bytes", head_size, group)
        if page_bytes == 0:
            raise ValueError(f"heads of {head_size} in groups of {group}: 32, 64 or 128 each, and no group larger than a head")
        if n_layer < 1 or n_kv_head < 1 or n_head % n_kv_head != 0 or n_head < 1:
            raise ValueError(f"{n_layer} layers of {n_head} heads over {n_kv_head}")
        if min(pages, requests, max_length) < 1 or pages * self.PAGE > 2**31 - 1 or max_length > 2**30:
            raise ValueError(f"{pages} pages of {self.PAGE} slots for {requests} requests of up to {max_length} tokens")
        self.device = torch.device("cuda", torch.cuda.current_device() if device.index is None else device.index)
        self._index = self.device.index
        self.n_layer, self.n_head, self.n_kv_head, self.head_size, self.group, self.dtype = n_layer, n_head, n_kv_head, head_size, group, dtype
        self.pages, self.requests, self.max_length, self.width = pages, requests, max_length, -(-max_length // self.PAGE)
        i32 = dict(dtype=torch.int32, device=self.device)
        self.blocks = torch.zeros((n_layer, pages, n_kv_head, page_bytes), dtype=torch.uint8, device=self.device)
        self.table = torch.full((requests, self.width), -1, **i32)
        self.lengths = torch.zeros(requests, **i32)
        self.free = torch.arange(pages - 1, -1, -1, **i32)
        self.n_free = torch.full((1,), pages, **i32)
        self._stamp = torch.zeros(requests, **i32)
        self.share = bool(share)
        self._shared = None                                               # a page's holders beyond the first, and scratch of -1
        if self.share:
            self._shared = torch.zeros((2, pages), **i32)
            self._shared[1].fill_(-1)
            self._shared_at = N.ptr(self._shared)
        self._none = torch.empty(0, dtype=dtype, device=self.device)      # (a result's type and device)
        self._code = N.dtype_code(dtype)
        self._struct = N.Kv4Cache(*(N.ptr(t) for t in (self.table, self.lengths, self.free, self.n_free, self._stamp)), requests, self.width, pages, max_length,
                                  n_head, n_kv_head, head_size, group, self._code)
        self._c = C.addressof(self._struct)
        self._layers = [N.ptr_at(self.blocks, i * self.blocks.stride(0)) for i in range(n_layer)]
        # (steps of requests that share pages are divided by groups that do)
        self._entry = {n: f"ll_kv4_{'shared_' if self.share else ''}{n}" for n in ("work_ints", "plan", "attn_scratch_bytes", "attn")}
        self._step = 0
        self._size_of = {}

    def _sizes(self, B: int, T: int, max_count: int) -> Tuple[int, int]:
        """Numbers of a plan's division, bytes of its attention's scratch."""
        key = (B, T, max_count)
        got = self._size_of.get(key)
        if got is None:
            if len(self._size_of) >= 256:      # (prompts come in many sizes)
                self._size_of.clear()
            got = self._size_of[key] = (N.call_ret(self._entry["work_ints"], self._c, *key), N.call_ret(self._entry["attn_scratch_bytes"], self._c, *key))
        return got

    def _here(self):
        """The cache's device as the current one, whose current stream the kernels go to."""
        return _NOTHING if _current_device() == self._index else torch.cuda.device(self.device)

    # ------------------------------------------------------------------ pages and slots
    def _whole(self, name: str, x: Whole) -> torch.Tensor:
        if not isinstance(x, torch.Tensor):
            x = torch.tensor(list(x), dtype=torch.int32, device=self.device)
        if x.dim() != 1 or x.dtype is not torch.int32 or x.get_device() != self._index:
            raise RuntimeError(f"{name}: int32 numbers on {self.device}, one for each sequence, not {x.dtype} {tuple(x.shape)} on {x.device}")
        return x.contiguous()

    def plan(self, rows: Whole, counts: Whole, tokens: int, *, max_count: Optional[int] = None) -> CachePlan:
        """Give the step's ``tokens`` rows their slots: the next ``counts[i]`` of them are sequence i's, the continuation of request ``rows[i]``.  A sequence
        may bring nothing; one that cannot be served is refused whole (``CachePlan.status``), its tokens get no slot and come out of ``attend`` as no numbers
        (of ``append`` too where it turns queries; else these are the caller's).  ``max_count``: the most that a sequence brings (``tokens`` unless said); it goes into the choice of kernels.
        Plans of earlier steps end with this one."""
        rows, counts = self._whole("rows", rows), self._whole("counts", counts)
        if rows.shape != counts.shape or rows.numel() == 0:
            raise RuntimeError(f"{rows.numel()} requests and {counts.numel()} counts")
        max_count = tokens if max_count is None else max_count
        if not 0 <= max_count or not 0 <= tokens < 2**31 // max(1, self.n_head):
            raise RuntimeError(f"a step of {tokens} tokens, {max_count} at most of a sequence")
        with self._here():
            self._step += 1
            plan = CachePlan(self, rows.numel(), tokens, min(max_count, tokens))
            N.call(self._entry["plan"], self._c, N.ptr(rows), N.ptr(counts), plan.B, tokens, plan.max_count, plan._out, plan._work, N.stream())
        return plan

    def truncate(self, rows: Whole, lengths: Whole) -> Optional[torch.Tensor]:
        """Cut request ``rows[i]`` to its first ``lengths[i]`` tokens (0 ends it); pages that no request needs any longer are free again.  Requests that are not
        longer stay as they are.  Where requests may share pages, a cut that ends inside a page which others hold takes a page for a copy of it; returned are then
        int32 numbers, one for each sequence: 0, or 1 where no page was free for that before the call and the request stays as it was."""
        rows, lengths = self._whole("rows", rows), self._whole("lengths", lengths)
        if rows.shape != lengths.shape or rows.numel() == 0:
            raise RuntimeError(f"{rows.numel()} requests and {lengths.numel()} lengths")
        with self._here():
            self._step += 1
            if self._shared is not None:
                return self._share("ll_kv4_release", rows, lengths)
            N.call("ll_kv4_truncate", self._c, N.ptr(rows), N.ptr(lengths), rows.numel(), N.stream())

    def fork(self, rows: Whole, into: Whole) -> torch.Tensor:
        """Make the empty requests ``into[i]`` copies of ``rows[i]``, one request of as many as one likes: they share its whole pages, and a last page that is not full is
        copied.  Returns int32 numbers, one for each sequence: 0; 1 where there is no free page for that; 3 where there is no such request, or ``into[i]`` is not
        empty or named before (``REASONS``).  Copies that are refused stay empty.  Plans of earlier steps end with this one."""
        if self._shared is None:
            raise RuntimeError("requests of this cache do not share pages: PagedCache4(.., share=True)")
        rows, into = self._whole("rows", rows), self._whole("into", into)
        if rows.shape != into.shape or rows.numel() == 0:
            raise RuntimeError(f"{rows.numel()} requests and {into.numel()} copies")
        with self._here():
            self._step += 1
            return self._share("ll_kv4_fork", rows, into)

    def _share(self, what: str, rows: torch.Tensor, other: torch.Tensor) -> torch.Tensor:
        B = rows.numel()
        out = self.lengths.new_empty(6 * B + 1)                              # statuses, and what the call notes of its sequences
        at = out.data_ptr()
        N.call(what, self._c, self._layers[0], self.n_layer, self._shared_at, rows.data_ptr(), other.data_ptr(), B, at, at + 4 * B, N.stream())
        return out[:B]

    def reset(self) -> None:
        """All requests end, and pages are given out as in the beginning."""
        self._step += 1
        self.table.fill_(-1)
        self.lengths.zero_()
        torch.arange(self.pages - 1, -1, -1, out=self.free)
        self.n_free.fill_(self.pages)
        if self._shared is not None:
            self._shared[0].zero_()

    # ------------------------------------------------------------------ a layer
    def _check(self, layer: int, plan: CachePlan) -> None:
        if not 0 <= layer < self.n_layer:
            raise RuntimeError(f"layer {layer} of {self.n_layer}")
        if plan.cache is not self or plan.step != self._step:
            raise RuntimeError("the plan is another cache's, or of a step before this cache's last plan, truncation or fork")

    def _rows(self, name: str, x: torch.Tensor, T: int, heads: int) -> Tuple[torch.Tensor, int]:
        """Rows as the kernels take them, and their distance: the heads of a token one after the other, tokens at any distance, 16-byte boundaries."""
        D = self.head_size
        if x.shape != (T, heads, D) or x.dtype is not self.dtype or x.get_device() != self._index:
            raise RuntimeError(f"{name}: {x.dtype} {tuple(x.shape)} on {x.device}, and the cache takes {self.dtype} {(T, heads, D)} on {self.device}")
        if x.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{name}: the 4-bit cache has no gradient")
        row, head, one = x.stride()
        if T < 2:                        # (one row's distance to a next one may be any)
            row = heads * D
        if one != 1 or (head != D and heads > 1) or row % 8 != 0 or row < heads * D or x.data_ptr() % 16 != 0:
            return x.clone(memory_format=torch.contiguous_format), heads * D
        return x, row

    def append(self, layer: int, plan: CachePlan, q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, rope: Optional[torch.Tensor] = None):
        """Round the step's keys and values ``[tokens, n_kv_head, head_size]`` into their slots.  With ``rope`` (fp32 ``[positions, head_size / 2, 2]``, as
        ``build_rope_cache``'s) keys are turned before, and queries ``[tokens, n_head, head_size]`` as well; returns the queries."""
        self._check(layer, plan)
        T = plan.T
        (k, k_row), (v, v_row) = self._rows("k", k, T, self.n_kv_head), self._rows("v", v, T, self.n_kv_head)
        out = q
        if rope is not None:
            if q is None:
                raise RuntimeError("queries have to be turned with their keys")
            q, q_row = self._rows("q", q, T, self.n_head)
            if rope.dtype is not torch.float32 or rope.dim() != 3 or rope.shape != (rope.shape[0], self.head_size // 2, 2) or not rope.is_contiguous() \
                    or rope.get_device() != self._index or rope.data_ptr() % 16 != 0:
                raise RuntimeError(f"rope: {rope.dtype} {tuple(rope.shape)} on {rope.device}, and the cache takes dense float32 [positions, {self.head_size // 2}, 2]")
            if rope.shape[0] < self.max_length:
                raise RuntimeError(f"rope: {rope.shape[0]} positions, and requests may have {self.max_length}")
            out = q.new_empty(T, self.n_head, self.head_size)
        if T == 0:
            return out
        with self._here():
            if rope is None:
                N.call("ll_kv4_append", self._c, self._layers[layer], None, 0, N.ptr(k), k_row, N.ptr(v), v_row, None, plan._positions, plan._slots, None, T,
                       N.stream())
            else:
                N.call("ll_kv4_append", self._c, self._layers[layer], N.ptr(q), q_row, N.ptr(k), k_row, N.ptr(v), v_row, N.ptr(rope), plan._positions,
                       plan._slots, N.ptr(out), T, N.stream())
        return out

    def read(self, layer: int, slots: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """What the cache holds at ``slots`` (a plan's, or any): keys and values ``[n, n_kv_head, head_size]``, no numbers for slots that there are not."""
        if not 0 <= layer < self.n_layer:
            raise RuntimeError(f"layer {layer} of {self.n_layer}")
        slots = self._whole("slots", slots)
        n = slots.numel()
        k = self._none.new_empty(n, self.n_kv_head, self.head_size)
        v = torch.empty_like(k)
        if n:
            with self._here():
                N.call("ll_kv4_read", self._c, self._layers[layer], N.ptr(slots), N.ptr(k), N.ptr(v), n, N.stream())
        return k, v

    def attend(self, layer: int, plan: CachePlan, q: torch.Tensor, scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Softmax attention of the step's queries ``[tokens, n_head, head_size]`` over what their requests hold up to their positions; the tokens' own keys
        have to be appended before.  ``scale`` of the scores: 1 / sqrt(head_size) unless given.  Rows of ``out`` behind the last token stay as they are; it may
        be ``q``."""
        self._check(layer, plan)
        T = plan.T
        q, q_row = self._rows("q", q, T, self.n_head)
        if out is None:
            out = q.new_empty(T, self.n_head, self.head_size)
        elif out.shape != q.shape or out.dtype != self.dtype or out.device != self.device or not out.is_contiguous() or out.data_ptr() % 16 != 0:
            raise RuntimeError(f"out: dense {self.dtype} {tuple(q.shape)} on {self.device}, not {out.dtype} {tuple(out.shape)} on {out.device}")
        scale = self.head_size ** -0.5 if scale is None else float(scale)
        if not 0 < scale < float("inf"):
            raise RuntimeError(f"scores times {scale}: more than 0")
        if T == 0:
            return out
        with self._here():
            scratch = self.blocks.new_empty(plan.scratch_bytes)
            N.call(self._entry["attn"], self._c, self._layers[layer], N.ptr(q), q_row, plan._work, N.ptr(out), plan.B, T, plan.max_count, scale, N.ptr(scratch), N.stream())
        return out
