"""KV pages held in 8 bits: typed wrappers over the flh_kv_* entry points of include/fuselink_hip.h (which states the
record of a page and every operator's definition).  The pages are ordinary pool pages to core.gather_pages and
core.scatter_pages, so a cache filled on one node moves and is read on another as it is.

Every call launches on `stream` (default: the current stream of the tensors' device) and returns at once; what it
allocates -- results that were not given, workspaces -- comes from that stream's pool.  A call that names a stream marks the
tensors given as used on it.  A workspace that is given belongs to one call at a time: calls on two streams, or two
graphs that may run at once, need one each.  What is wrong with device-resident page numbers, lengths and starts shows as
FLH_E_RANGE in `status` (core.new_status()).

Results that were not given hold nothing defined in the rows of tokens that are no sequence's.

No operator has a gradient: where gradients are recorded, tensors that require one are refused.  What a call writes (pages, outputs
and weights given, status) is written behind autograd's back, without a new version of the tensor."""
from __future__ import annotations

import contextlib
import ctypes as C
import math
import struct
from typing import Optional

import torch

from . import _lib
from ._lib import KvAttendParams, KvEvictParams, KvSelectParams, KvStoreParams, check

TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_I32, _F32 = torch.int32, torch.float32

# The parameter blocks as struct formats: filling a ctypes structure field by field took longer than the launch.
_CACHE, _SEQS = "QQIIII", "QQQQIIII"
_STORE = struct.Struct("=" + _CACHE + _SEQS + "QQ" + "QQQQ" + "II" + "Q")
_ATTEND = struct.Struct("=" + _CACHE + _SEQS + "QQ" + "QQQQ" + "Q" + "IIfI" + "QQQ" + "QQQQ" + "II" + "QQQ")
_SELECT = struct.Struct("=" + _CACHE + _SEQS + "Q" + "QQ" + "IIIIII" + "Q" + "QQQ")
_EVICT = struct.Struct("=" + _CACHE + _CACHE + _SEQS + "QQ" + "QQQ" + "QQQ" + "QQ" + "IIIIII" + "Q")
for _f, _c in ((_STORE, KvStoreParams), (_ATTEND, KvAttendParams), (_SELECT, KvSelectParams), (_EVICT, KvEvictParams)):
    assert _f.size == C.sizeof(_c), _c


def page_bytes(tokens: int, heads: int, dim: int) -> int:
    """Bytes of the record of a page: codes, key bounds and scales, rounded up to 128."""
    return int(_lib.load().flh_kv_page_bytes(tokens, heads, dim))


class PageCache:
    """A pool of page records: `pages` is a uint8 device tensor [n_pages, >= page_bytes], its rows a multiple of 16
    bytes apart (a slice of a wider pool -- one layer of several -- will do)."""

    def __init__(self, pages: torch.Tensor, tokens: int, heads: int, dim: int):
        _need(pages.dim() == 2 and pages.dtype == torch.uint8 and pages.stride(1) == 1, "pages must be a uint8 tensor [n_pages, bytes]")
        _need(0 < tokens <= 256 and tokens % 16 == 0, f"{tokens} tokens a page (a multiple of 16, up to 256)")
        _need(0 < dim <= 256 and dim % 16 == 0, f"head dim {dim} (a multiple of 16, up to 256)")
        _need(0 < heads <= 1024, f"{heads} heads (1..1024)")
        _need(pages.shape[0] > 0, "a pool of no pages")
        need = page_bytes(tokens, heads, dim)
        stride = pages.stride(0) if pages.shape[0] > 1 else (pages.shape[1] + 15) // 16 * 16   # one page: the stride is never used
        _need(pages.shape[1] >= need and stride >= need and stride % 16 == 0 and pages.data_ptr() % 16 == 0,
              f"records of {need} bytes in rows of {pages.shape[1]}, {stride} apart")
        self.pages, self.tokens, self.heads, self.dim = pages, tokens, heads, dim
        self.c = (pages.data_ptr(), stride, pages.shape[0], tokens, heads, dim)
        self.device, self.index = pages.device, pages.get_device()

    def codes(self):
        """K and V codes, float8_e4m3fn views [n_pages, heads, tokens, dim] of the pool."""
        n, a = self.pages.shape[0], self.heads * self.tokens * self.dim
        return tuple(self.pages[:, i * a:(i + 1) * a].view(torch.float8_e4m3fn).unflatten(1, (self.heads, self.tokens, self.dim)) for i in (0, 1))

    def bounds(self):
        """low and high, int8 views [n_pages, heads, dim]."""
        a, m = 2 * self.heads * self.tokens * self.dim, self.heads * self.dim
        return tuple(self.pages[:, a + i * m:a + (i + 1) * m].view(torch.int8).unflatten(1, (self.heads, self.dim)) for i in (0, 1))

    def scales(self):
        """Scales of K and of V, a float32 view [n_pages, heads, 2]."""
        a = 2 * self.heads * self.dim * (self.tokens + 1)
        return self.pages[:, a:a + 8 * self.heads].view(torch.float32).unflatten(1, (self.heads, 2))


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _wrong(cache: PageCache, name: str, t, what: str) -> None:
    _need(cache.index >= 0, "the pool must be on a GPU: there is no CPU path")
    raise ValueError(f"{name}: {what}, its last dimension contiguous, on {cache.device}; not {tuple(t.shape)} {t.dtype}, strides {t.stride()}, on {t.device}")


def _check(cache: PageCache, name: str, t: torch.Tensor, dtype, dims: int):
    """Shape and strides of a tensor that is what it has to be."""
    shape, stride = t.shape, t.stride()
    if t.dtype is not dtype or len(shape) != dims or (stride[-1] != 1 and shape[-1] > 1) or t.get_device() != cache.index:
        _wrong(cache, name, t, f"{dims} dimensions of {dtype}")
    return shape, stride


def _no_gradient(*tensors) -> None:
    for t in tensors:
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise ValueError("the operators on KV pages have no gradient: detach what requires one, or call them under torch.no_grad()")


def _check_written(name: str, t: torch.Tensor) -> None:
    if any(n > 1 and st == 0 for n, st in zip(t.shape, t.stride())):
        raise ValueError(f"{name}: written, but some of its elements share memory")


def _apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    """No element of one is an element of the other: their extents are disjoint, or rows a common stride apart lie between each other."""
    if a.numel() == 0 or b.numel() == 0:
        return True
    inner = [t.element_size() * (1 + sum((n - 1) * st for n, st in zip(t.shape[1:], t.stride()[1:]))) for t in (a, b)]
    pa, pb = a.data_ptr(), b.data_ptr()
    row = a.stride(0) * a.element_size()
    if pa + (a.shape[0] - 1) * row + inner[0] <= pb or pb + (b.shape[0] - 1) * b.stride(0) * b.element_size() + inner[1] <= pa:
        return True
    if row == 0 or row != b.stride(0) * b.element_size():
        return False
    d = (pb - pa) % row
    return d >= inner[0] and row - d >= inner[1]


def _seqs(cache: PageCache, table, lens, status, starts, n_tokens: int):
    """The fields of flh_kv_seqs, and the status word's address."""
    _need(cache.index >= 0, "the pool must be on a GPU: there is no CPU path")
    (n, width), (stride, _) = _check(cache, "page_table", table, _I32, 2)
    (n_lens,), _ = _check(cache, "lens", lens, _I32, 1)
    (words,), _ = _check(cache, "status", status, _I32, 1)
    if n == 1:
        stride = width
    if not (n > 0 and width > 0 and n_lens == n and stride >= width and words > 0):
        raise ValueError(f"page_table of {tuple(table.shape)} (rows {stride} apart) for {n_lens} lens, {words} words of status")
    if starts is not None:
        (n_starts,), _ = _check(cache, "starts", starts, _I32, 1)
        if n_starts != n + 1:
            raise ValueError(f"{n_starts} starts for {n} sequences (one more than sequences)")
        sp = starts.data_ptr()
    else:
        if n_tokens % n:
            raise ValueError(f"{n_tokens} tokens do not divide into {n} sequences; give starts")
        sp = 0
    return (sp, lens.data_ptr(), table.data_ptr(), stride, width, n, n_tokens, 0), status.data_ptr()


def _queries(cache: PageCache, q: torch.Tensor):
    """Tokens, query heads, strides and type of the queries."""
    if q.dtype is not torch.bfloat16 and q.dtype is not torch.float16:
        _wrong(cache, "q", q, "bf16 or fp16")
    (n, hq, d), (st, sh, _) = _check(cache, "q", q, q.dtype, 3)
    if d != cache.dim or hq == 0 or hq % cache.heads:
        raise ValueError(f"q {tuple(q.shape)} over {cache.heads} heads of {cache.dim}")
    return n, hq, st, sh, 0 if q.dtype is torch.bfloat16 else 1


class _On:
    """Device and stream of a call that names a stream, or whose tensors are not on the current device: allocations inside belong
    to the stream, and the tensors given (all found sound by then) are marked as used on it."""

    def __init__(self, cache: PageCache, stream: Optional[torch.cuda.Stream], *tensors):
        _need(stream is None or stream.device == cache.device, f"stream of {stream and stream.device}, tensors of {cache.device}")
        self.cache, self.stream, self.tensors, self.stack = cache, stream, tensors, contextlib.ExitStack()

    def __enter__(self):
        if self.stream is None:
            self.stack.enter_context(torch.cuda.device(self.cache.device))
            return torch.cuda.current_stream(self.cache.device).cuda_stream
        with contextlib.ExitStack() as stack:      # (undone if anything below raises)
            stack.enter_context(torch.cuda.stream(self.stream))
            if not torch.cuda.is_current_stream_capturing():
                for t in self.tensors:
                    if t is not None:
                        t.record_stream(self.stream)
            self.stack = stack.pop_all()
        return self.stream.cuda_stream

    def __exit__(self, *exc):
        self.stack.close()


class _Here:
    """The current stream of the current device."""

    def __init__(self, index: int):
        self.ptr = torch._C._cuda_getCurrentRawStream(index)

    def __enter__(self):
        return self.ptr

    def __exit__(self, *exc):
        pass


def _on(cache: PageCache, stream, *tensors):
    if stream is None and torch.cuda.current_device() == cache.index:
        return _Here(cache.index)
    return _On(cache, stream, *tensors)


def _check_workspace(cache: PageCache, given: Optional[torch.Tensor], need: int) -> Optional[torch.Tensor]:
    """The workspace that the caller gives, if the call needs one."""
    if given is None or need == 0:
        return None
    _need(given.get_device() == cache.index and given.is_contiguous() and given.numel() * given.element_size() >= need and given.data_ptr() % 16 == 0,
          f"workspace: {need} contiguous bytes on {cache.device}, 16-byte aligned")
    return given


def _workspace(cache: PageCache, given: Optional[torch.Tensor], need: int):
    """Address and bytes of a workspace, and what owns it."""
    if need == 0:
        return 0, 0, None
    if given is None:
        given = torch.empty(need, dtype=torch.uint8, device=cache.device)
    return given.data_ptr(), given.numel() * given.element_size(), given


def store(cache: PageCache, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, lens: torch.Tensor, status: torch.Tensor, *,
          starts: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None) -> None:
    """flh_kv_store: appends k and v [n_tokens, heads, dim] (bf16, fp16 or fp32) to sequences that hold `lens` tokens
    before the call.  `starts` [n_seqs + 1] says whose tokens are whose; without it every sequence has equally many."""
    _no_gradient(k, v)
    kind = TYPES.get(k.dtype)
    if kind is None:
        _wrong(cache, "k", k, "bf16, fp16 or fp32")
    shape, (kt, kh, _) = _check(cache, "k", k, k.dtype, 3)
    v_shape, (vt, vh, _) = _check(cache, "v", v, k.dtype, 3)
    if shape != v_shape or shape[1] != cache.heads or shape[2] != cache.dim:
        raise ValueError(f"k {tuple(shape)} and v {tuple(v_shape)} for {cache.heads} heads of {cache.dim}")
    seqs, word = _seqs(cache, page_table, lens, status, starts, shape[0])
    p = _STORE.pack(*cache.c, *seqs, k.data_ptr(), v.data_ptr(), kt, kh, vt, vh, kind, 0, word)
    with _on(cache, stream, cache.pages, k, v, page_table, lens, status, starts) as sp:
        check(_lib.load().flh_kv_store(p, sp))


def attend(cache: PageCache, q: torch.Tensor, page_table: torch.Tensor, lens: torch.Tensor, status: torch.Tensor, *,
           starts: Optional[torch.Tensor] = None, scale: Optional[float] = None, causal: bool = True, out: Optional[torch.Tensor] = None,
           lse: Optional[torch.Tensor] = None, selected: Optional[torch.Tensor] = None, weights: Optional[torch.Tensor] = None,
           weights_in: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None,
           stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """flh_kv_attend: attention of q [n_tokens, q_heads, dim] (bf16 or fp16) over the `lens` tokens of their sequences,
    those of the call included (store them first).  `scale` defaults to 1 / sqrt(dim).  `lse` (float32 [n_tokens, q_heads],
    contiguous) receives the logarithms of the rows' sums.  `selected` (from select_pages) restricts every query token and head to
    those pages.  `weights` (float32 [n_seqs, heads, positions]) gains what attention every key drew: it is added to in
    place, or written as `weights_in` plus the gain when that is given."""
    _no_gradient(q, out, lse, weights, weights_in)
    n, hq, qt, qh, kind = _queries(cache, q)
    seqs, word = _seqs(cache, page_table, lens, status, starts, n)
    n_seqs, heads = seqs[5], cache.heads
    lse_p = sel_p = count = win_p = w_p = wis = wih = ws = wh = width = 0
    if lse is not None:
        shape, _ = _check(cache, "lse", lse, _F32, 2)
        _need(lse.is_contiguous() and shape == q.shape[:2], f"lse: contiguous {tuple(q.shape[:2])}")
        lse_p = lse.data_ptr()
    if selected is not None:
        (a, b, count), _ = _check(cache, "selected", selected, _I32, 3)
        _need(weights is None, "weights are kept over all pages, not over selected ones")
        _need(a == n and b == heads and count > 0 and selected.is_contiguous(), f"selected: contiguous [{n}, {heads}, pages]")
        sel_p = selected.data_ptr()
    if weights is not None:
        (a, b, width), (ws, wh, _) = _check(cache, "weights", weights, _F32, 3)
        _need(a == n_seqs and b == heads and width > 0, f"weights: [{n_seqs}, {heads}, positions]")
        _check_written("weights", weights)
        w_p, win_p, wis, wih = weights.data_ptr(), weights.data_ptr(), ws, wh
        if weights_in is not None:
            shape, (wis, wih, _) = _check(cache, "weights_in", weights_in, _F32, 3)
            _need(shape == weights.shape, f"weights_in: [{n_seqs}, {heads}, {width}]")
            win_p = weights_in.data_ptr()
            _need((win_p == w_p and (wis, wih) == (ws, wh)) or _apart(weights, weights_in), "weights and weights_in overlap without being the same")
    else:
        _need(weights_in is None, "weights_in without weights")
    if out is not None:
        _check(cache, "out", out, q.dtype, 3)
        _check_written("out", out)
        _need(out.shape == q.shape, f"out {tuple(out.shape)} for q {tuple(q.shape)}")
        _need(_apart(out, q), "out overlaps q")
    lib = _lib.load()

    def block(out_p, ot, oh, wp, wb):
        return _ATTEND.pack(*cache.c, *seqs, q.data_ptr(), out_p, qt, qh, ot, oh, lse_p, kind, hq, 1.0 / math.sqrt(cache.dim) if scale is None else scale,
                            1 if causal else 0, sel_p, win_p, w_p, wis, wih, ws, wh, count, width, wp, wb, word)

    sizes = (cache.c[3:], seqs[4:7], seqs[0] != 0, hq, count, w_p != 0)
    need = _needs.get(sizes)
    if need is None:
        if len(_needs) >= 4096:
            _needs.clear()
        need = _needs[sizes] = check(lib.flh_kv_attend_workspace_bytes(block(0, 0, 0, 0, 0)))
    workspace = _check_workspace(cache, workspace, need)
    with _on(cache, stream, cache.pages, q, page_table, lens, status, starts, lse, selected, weights, weights_in, out, workspace) as sp:
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        ot, oh, _ = out.stride()
        wp, wb, owner = _workspace(cache, workspace, need)
        check(lib.flh_kv_attend(block(out.data_ptr(), ot, oh, wp, wb), sp))
    return out


_needs: dict = {}    # sizes of a call -> bytes of its workspace


def select_pages(cache: PageCache, q: torch.Tensor, page_table: torch.Tensor, lens: torch.Tensor, count: int, status: torch.Tensor, *,
                 starts: Optional[torch.Tensor] = None, first: int = 1, last: int = 1, causal: bool = True, out: Optional[torch.Tensor] = None,
                 workspace: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """flh_kv_select: for every query token and key-value head the `count` pages (int32 [n_tokens, heads, count], ascending, -1 behind
    them) whose keys may weigh most, the first `first` and last `last` ones always among them."""
    n, hq, qt, qh, kind = _queries(cache, q)
    _need(0 < count < 2 ** 31 and first >= 0 and last >= 0 and first + last <= count, f"{count} pages with {first} first and {last} last ones")
    seqs, word = _seqs(cache, page_table, lens, status, starts, n)
    if out is not None:
        shape, _ = _check(cache, "out", out, _I32, 3)
        _need(out.is_contiguous() and tuple(shape) == (n, cache.heads, count), f"out: contiguous [{n}, {cache.heads}, {count}]")
    need = 4 * n * cache.heads * seqs[4]         # flh_kv_select_workspace_bytes
    workspace = _check_workspace(cache, workspace, need)
    with _on(cache, stream, cache.pages, q, page_table, lens, status, starts, out, workspace) as sp:
        if out is None:
            out = torch.empty((n, cache.heads, count), dtype=_I32, device=cache.device)
        wp, wb, owner = _workspace(cache, workspace, need)
        check(_lib.load().flh_kv_select(_SELECT.pack(*cache.c, *seqs, q.data_ptr(), qt, qh, kind, hq, count, first, last, 1 if causal else 0,
                                                     out.data_ptr(), wp, wb, word), sp))
    return out


def evict(cache: PageCache, page_table: torch.Tensor, lens: torch.Tensor, weights: torch.Tensor, budget: int, to: PageCache, to_table: torch.Tensor,
          status: torch.Tensor, *, first: int = 0, recent: int = 0, kept: Optional[torch.Tensor] = None, new_weights: Optional[torch.Tensor] = None,
          new_lens: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None):
    """flh_kv_evict: cuts every sequence back to `budget` tokens a head -- the first `first`, the last `recent` and those of the largest
    `weights` [n_seqs, heads, positions] -- packed into the pages of `to` that `to_table` [n_seqs, pages] names, none of which may be
    among those that are read.  Returns (kept, new_weights, new_lens): positions [n_seqs, heads, budget] with -1 behind
    them, the weights kept with zeros behind them ([n_seqs, heads, >= budget]), and the new lengths (`new_lens` is other memory than `lens`)."""
    _no_gradient(weights, new_weights)
    seqs, word = _seqs(cache, page_table, lens, status, None, 0)
    b, h = seqs[5], cache.heads
    _need(to.index == cache.index and to.heads == h and to.dim == cache.dim, "the new cache differs in device, heads or head dim")
    (wb, wh, width), (ws_s, ws_h, _) = _check(cache, "weights", weights, _F32, 3)
    _need(wb == b and wh == h and width > 0, f"weights: [{b}, {h}, positions]")
    _need(0 < budget <= 1 << 30 and first >= 0 and recent >= 0 and first + recent <= budget, f"a budget of {budget} with {first} first and {recent} recent tokens")
    (tb, to_width), (stride, _) = _check(cache, "to_table", to_table, _I32, 2)
    if b == 1:
        stride = to_width
    _need(tb == b and to_width >= (budget + to.tokens - 1) // to.tokens and stride >= to_width, f"to_table: [{b}, >= {(budget + to.tokens - 1) // to.tokens}]")
    _need(to_table.data_ptr() != page_table.data_ptr() or to.c[0] != cache.c[0], "to_table is page_table: the new pages must not be among those that are read")
    if kept is not None:
        shape, _ = _check(cache, "kept", kept, _I32, 3)
        _need(kept.is_contiguous() and tuple(shape) == (b, h, budget), f"kept: contiguous [{b}, {h}, {budget}]")
    if new_weights is not None:
        (nb, nhh, nw), (ns, nh, _) = _check(cache, "new_weights", new_weights, _F32, 3)
        _check_written("new_weights", new_weights)
        _need(nb == b and nhh == h and nw >= budget, f"new_weights: [{b}, {h}, >= {budget}]")
        _need(_apart(new_weights, weights), "new_weights overlaps weights")
    else:
        ns, nh, nw = h * budget, budget, budget
    if new_lens is not None:
        (nl,), _ = _check(cache, "new_lens", new_lens, _I32, 1)
        _check_written("new_lens", new_lens)
        _need(nl == b, f"new_lens: [{b}]")
        _need(_apart(new_lens, lens), "new_lens overlaps lens")
    with _on(cache, stream, cache.pages, to.pages, page_table, lens, weights, to_table, status, kept, new_weights, new_lens) as sp:
        if kept is None:
            kept = torch.empty((b, h, budget), dtype=_I32, device=cache.device)
        if new_weights is None:
            new_weights = torch.empty((b, h, budget), dtype=_F32, device=cache.device)
        if new_lens is None:
            new_lens = torch.empty(b, dtype=_I32, device=cache.device)
        check(_lib.load().flh_kv_evict(_EVICT.pack(*cache.c, *to.c, *seqs, to_table.data_ptr(), stride, weights.data_ptr(), ws_s, ws_h,
                                                   new_weights.data_ptr(), ns, nh, kept.data_ptr(), new_lens.data_ptr(), to_width, width, nw,
                                                   budget, first, recent, word), sp))
    return kept, new_weights, new_lens
