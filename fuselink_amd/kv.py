"""KV pages held in 8 bits: typed wrappers over the flh_kv_* entry points of include/fuselink_hip.h (which states the
record of a page and every operator's definition).  The pages are ordinary pool pages to core.gather_pages and
core.scatter_pages, so a cache filled on one node moves and is read on another as it is.

Every call launches on `stream` (default: the current stream of the tensors' device) and returns at once; what it
allocates -- results that were not given, workspaces -- comes from that stream's pool.  Tensors that belong to another
stream are marked as used on this one.  What is wrong with device-resident page numbers, lengths and starts shows as
FLH_E_RANGE in `status` (core.new_status())."""
from __future__ import annotations

import contextlib
import ctypes as C
import math
from typing import Optional

import torch

from . import _lib
from ._lib import KvAttendParams, KvCache, KvEvictParams, KvSelectParams, KvSeqs, KvStoreParams, check

TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


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
        self.c = KvCache(pages.data_ptr(), stride, pages.shape[0], tokens, heads, dim)

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


def _check(dev: torch.device, name: str, t: torch.Tensor, dtype, dims: int) -> None:
    if t.device != dev or t.dim() != dims or (t.dtype != dtype if dtype is not None else t.dtype not in TYPES) or (t.shape[-1] > 1 and t.stride(-1) != 1):
        raise ValueError(f"{name}: a tensor of {dims} dimensions on {dev}, {dtype or 'bf16, fp16 or fp32'}, its last dimension contiguous; "
                         f"not {tuple(t.shape)} {t.dtype} on {t.device}")


def _check_written(name: str, t: torch.Tensor) -> None:
    if any(n > 1 and st == 0 for n, st in zip(t.shape, t.stride())):
        raise ValueError(f"{name}: written, but some of its elements share memory")


def _seqs(cache: PageCache, table, lens, status, starts, n_tokens: int) -> KvSeqs:
    dev = cache.pages.device
    _need(dev.type == "cuda", "the pool must be on a GPU: there is no CPU path")
    _check(dev, "page_table", table, torch.int32, 2)
    _check(dev, "lens", lens, torch.int32, 1)
    _check(dev, "status", status, torch.int32, 1)
    _need(status.numel() >= 1, "status: one word at least")
    n = table.shape[0]
    _need(n > 0 and table.shape[1] > 0 and lens.shape[0] == n, f"page_table of {tuple(table.shape)} for {lens.shape[0]} lens")
    stride = table.stride(0) if n > 1 else table.shape[1]
    _need(stride >= table.shape[1], "page_table: its rows overlap")
    if starts is not None:
        _check(dev, "starts", starts, torch.int32, 1)
        _need(starts.shape[0] == n + 1, f"{starts.shape[0]} starts for {n} sequences (one more than sequences)")
        sp = starts.data_ptr()
    else:
        _need(n_tokens % n == 0, f"{n_tokens} tokens do not divide into {n} sequences; give starts")
        sp = None
    return KvSeqs(sp, lens.data_ptr(), table.data_ptr(), stride, table.shape[1], n, n_tokens, 0)


class _On:
    """Device and stream of a call: allocations inside belong to the stream, tensors given are marked as used on it."""

    def __init__(self, dev: torch.device, stream: Optional[torch.cuda.Stream], *tensors):
        self.stack = None
        if stream is None:
            if torch.cuda.current_device() != dev.index:
                self.stack = contextlib.ExitStack()
                self.stack.enter_context(torch.cuda.device(dev))
            self.ptr = C.c_void_p(torch._C._cuda_getCurrentRawStream(dev.index))
            return
        _need(stream.device == dev, f"stream of {stream.device}, tensors of {dev}")
        self.stack = contextlib.ExitStack()
        self.stack.enter_context(torch.cuda.stream(stream))
        self.ptr = C.c_void_p(stream.cuda_stream)
        if not torch.cuda.is_current_stream_capturing():
            for t in tensors:
                if t is not None:
                    t.record_stream(stream)

    def __enter__(self):
        return self.ptr

    def __exit__(self, *exc):
        if self.stack is not None:
            self.stack.close()


def _workspace(given: Optional[torch.Tensor], need: int, dev: torch.device) -> Optional[torch.Tensor]:
    if need == 0:
        return None
    if given is None:
        return torch.empty(need, dtype=torch.uint8, device=dev)
    nbytes = given.numel() * given.element_size()
    _need(given.device == dev and given.is_contiguous() and nbytes >= need and given.data_ptr() % 16 == 0, f"workspace: {need} contiguous bytes on {dev}, 16-byte aligned")
    return given


def store(cache: PageCache, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, lens: torch.Tensor, status: torch.Tensor, *,
          starts: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None) -> None:
    """flh_kv_store: appends k and v [n_tokens, heads, dim] (bf16, fp16 or fp32) to sequences that hold `lens` tokens
    before the call.  `starts` [n_seqs + 1] says whose tokens are whose; without it every sequence has equally many."""
    dev = cache.pages.device
    _check(dev, "k", k, None, 3)
    _check(dev, "v", v, k.dtype, 3)
    _need(k.shape == v.shape and tuple(k.shape[1:]) == (cache.heads, cache.dim), f"k {tuple(k.shape)} and v {tuple(v.shape)} for {cache.heads} heads of {cache.dim}")
    p = KvStoreParams(cache.c, _seqs(cache, page_table, lens, status, starts, k.shape[0]), k.data_ptr(), v.data_ptr(),
                      k.stride(0), k.stride(1), v.stride(0), v.stride(1), TYPES[k.dtype], 0, status.data_ptr())
    with _On(dev, stream, cache.pages, k, v, page_table, lens, status, starts) as sp:
        check(_lib.load().flh_kv_store(C.byref(p), sp))


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
    dev = cache.pages.device
    _check(dev, "q", q, None, 3)
    _need(q.dtype != torch.float32, "q: bf16 or fp16")
    n, hq = q.shape[0], q.shape[1]
    _need(q.shape[2] == cache.dim and hq > 0 and hq % cache.heads == 0, f"q {tuple(q.shape)} over {cache.heads} heads of {cache.dim}")
    s = _seqs(cache, page_table, lens, status, starts, n)
    p = KvAttendParams()
    if lse is not None:
        _check(dev, "lse", lse, torch.float32, 2)
        _need(lse.is_contiguous() and lse.shape == q.shape[:2], f"lse: contiguous {tuple(q.shape[:2])}")
        p.d_lse = lse.data_ptr()
    if selected is not None:
        _check(dev, "selected", selected, torch.int32, 3)
        _need(selected.is_contiguous() and tuple(selected.shape[:2]) == (n, cache.heads), f"selected: contiguous [{n}, {cache.heads}, pages]")
        _need(weights is None, "weights are kept over all pages, not over selected ones")
        _need(selected.shape[2] > 0, "selected: no pages")
        p.d_selected, p.n_selected = selected.data_ptr(), min(selected.shape[2], 0xffffffff)
    if weights_in is not None:
        _need(weights is not None, "weights_in without weights")
    if weights is not None:
        src = weights if weights_in is None else weights_in
        for name, w in (("weights", weights), ("weights_in", src)):
            _check(dev, name, w, torch.float32, 3)
            _need(tuple(w.shape[:2]) == (s.n_seqs, cache.heads) and w.shape == weights.shape and w.shape[2] > 0, f"{name}: [{s.n_seqs}, {cache.heads}, positions]")
        _check_written("weights", weights)
        p.d_weights, p.d_weights_in, p.weights_width = weights.data_ptr(), src.data_ptr(), weights.shape[2]
        p.weights_seq_stride, p.weights_head_stride = weights.stride(0), weights.stride(1)
        p.weights_in_seq_stride, p.weights_in_head_stride = src.stride(0), src.stride(1)
    p.cache, p.seqs = cache.c, s
    p.d_q, p.q_token_stride, p.q_head_stride = q.data_ptr(), q.stride(0), q.stride(1)
    p.type, p.q_heads, p.causal, p.d_status = TYPES[q.dtype], hq, int(causal), status.data_ptr()
    p.scale = 1.0 / math.sqrt(cache.dim) if scale is None else scale
    lib = _lib.load()
    with _On(dev, stream, cache.pages, q, page_table, lens, status, starts, lse, selected, weights, weights_in, out, workspace) as sp:
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        else:
            _check(dev, "out", out, q.dtype, 3)
            _check_written("out", out)
            _need(out.shape == q.shape, f"out {tuple(out.shape)} for q {tuple(q.shape)}")
        p.d_out, p.out_token_stride, p.out_head_stride = out.data_ptr(), out.stride(0), out.stride(1)
        need = check(lib.flh_kv_attend_workspace_bytes(C.byref(p)))
        if need:
            workspace = _workspace(workspace, need, dev)
            p.d_workspace, p.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        check(lib.flh_kv_attend(C.byref(p), sp))
    return out


def select_pages(cache: PageCache, q: torch.Tensor, page_table: torch.Tensor, lens: torch.Tensor, count: int, status: torch.Tensor, *,
                 starts: Optional[torch.Tensor] = None, first: int = 1, last: int = 1, causal: bool = True, out: Optional[torch.Tensor] = None,
                 workspace: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """flh_kv_select: for every query token and key-value head the `count` pages (int32 [n_tokens, heads, count], ascending, -1 behind
    them) whose keys may weigh most, the first `first` and last `last` ones always among them."""
    dev = cache.pages.device
    _check(dev, "q", q, None, 3)
    _need(q.dtype != torch.float32, "q: bf16 or fp16")
    n, hq = q.shape[0], q.shape[1]
    _need(q.shape[2] == cache.dim and hq > 0 and hq % cache.heads == 0, f"q {tuple(q.shape)} over {cache.heads} heads of {cache.dim}")
    _need(0 < count < 2 ** 31 and first >= 0 and last >= 0 and first + last <= count, f"{count} pages with {first} first and {last} last ones")
    s = _seqs(cache, page_table, lens, status, starts, n)
    lib = _lib.load()
    with _On(dev, stream, cache.pages, q, page_table, lens, status, starts, out, workspace) as sp:
        if out is None:
            out = torch.empty((n, cache.heads, count), dtype=torch.int32, device=dev)
        else:
            _check(dev, "out", out, torch.int32, 3)
            _need(out.is_contiguous() and tuple(out.shape) == (n, cache.heads, count), f"out: contiguous [{n}, {cache.heads}, {count}]")
        workspace = _workspace(workspace, int(lib.flh_kv_select_workspace_bytes(n, cache.heads, s.table_width)), dev)
        p = KvSelectParams(cache.c, s, q.data_ptr(), q.stride(0), q.stride(1), TYPES[q.dtype], hq, count, first, last, int(causal), out.data_ptr(),
                           workspace.data_ptr() if workspace is not None else None,
                           workspace.numel() * workspace.element_size() if workspace is not None else 0, status.data_ptr())
        check(lib.flh_kv_select(C.byref(p), sp))
    return out


def evict(cache: PageCache, page_table: torch.Tensor, lens: torch.Tensor, weights: torch.Tensor, budget: int, to: PageCache, to_table: torch.Tensor,
          status: torch.Tensor, *, first: int = 0, recent: int = 0, kept: Optional[torch.Tensor] = None, new_weights: Optional[torch.Tensor] = None,
          new_lens: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None):
    """flh_kv_evict: cuts every sequence back to `budget` tokens a head -- the first `first`, the last `recent` and those of the largest
    `weights` [n_seqs, heads, positions] -- packed into the pages of `to` that `to_table` [n_seqs, pages] names, none of which may be
    among those that are read.  Returns (kept, new_weights, new_lens): positions [n_seqs, heads, budget] with -1 behind
    them, the weights kept with zeros behind them ([n_seqs, heads, >= budget]), and the new lengths."""
    dev = cache.pages.device
    s = _seqs(cache, page_table, lens, status, None, 0)
    b, h = s.n_seqs, cache.heads
    _need(to.pages.device == dev and to.heads == h and to.dim == cache.dim, "the new cache differs in device, heads or head dim")
    _check(dev, "weights", weights, torch.float32, 3)
    _need(tuple(weights.shape[:2]) == (b, h) and weights.shape[2] > 0, f"weights: [{b}, {h}, positions]")
    _need(0 < budget <= 1 << 30 and first >= 0 and recent >= 0 and first + recent <= budget, f"a budget of {budget} with {first} first and {recent} recent tokens")
    _check(dev, "to_table", to_table, torch.int32, 2)
    per = (budget + to.tokens - 1) // to.tokens
    stride = to_table.stride(0) if b > 1 else to_table.shape[1]
    _need(to_table.shape[0] == b and to_table.shape[1] >= per and stride >= to_table.shape[1], f"to_table: [{b}, >= {per}]")
    with _On(dev, stream, cache.pages, to.pages, page_table, lens, weights, to_table, status, kept, new_weights, new_lens) as sp:
        if kept is None:
            kept = torch.empty((b, h, budget), dtype=torch.int32, device=dev)
        if new_weights is None:
            new_weights = torch.empty((b, h, budget), dtype=torch.float32, device=dev)
        if new_lens is None:
            new_lens = torch.empty(b, dtype=torch.int32, device=dev)
        _check(dev, "kept", kept, torch.int32, 3)
        _check(dev, "new_weights", new_weights, torch.float32, 3)
        _check(dev, "new_lens", new_lens, torch.int32, 1)
        _need(kept.is_contiguous() and tuple(kept.shape) == (b, h, budget), f"kept: contiguous [{b}, {h}, {budget}]")
        _need(tuple(new_weights.shape[:2]) == (b, h) and new_weights.shape[2] >= budget, f"new_weights: [{b}, {h}, >= {budget}]")
        _check_written("new_weights", new_weights)
        _need(new_lens.shape[0] == b, f"new_lens: [{b}]")
        p = KvEvictParams(cache.c, to.c, s, to_table.data_ptr(), stride, weights.data_ptr(), weights.stride(0), weights.stride(1),
                          new_weights.data_ptr(), new_weights.stride(0), new_weights.stride(1), kept.data_ptr(), new_lens.data_ptr(),
                          to_table.shape[1], weights.shape[2], new_weights.shape[2], budget, first, recent, status.data_ptr())
        check(_lib.load().flh_kv_evict(C.byref(p), sp))
    return kept, new_weights, new_lens
