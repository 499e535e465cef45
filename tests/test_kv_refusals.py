"""Calls on KV pages that are refused before anything is launched (no GPU needed: no kernel is reached)."""
import ctypes as C
import os

import pytest
import torch

from fuselink_amd import _lib, kv

E_ARG = -1
P = 1 << 20            # stands for a device pointer: refused calls never follow it


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def cache(**kw):
    c = _lib.KvCache(P, 34944, 8, 16, 8, 128)
    for n, v in kw.items():
        setattr(c, n, v)
    return c


def seqs(**kw):
    s = _lib.KvSeqs(None, P, P, 4, 4, 2, 2, 0)
    for n, v in kw.items():
        setattr(s, n, v)
    return s


def store(c=None, s=None, **kw):
    p = _lib.KvStoreParams(c or cache(), s or seqs(), P, P, 1024, 128, 1024, 128, 0, 0, P)
    for n, v in kw.items():
        setattr(p, n, v)
    return p


def attend(c=None, s=None, **kw):
    p = _lib.KvAttendParams(cache=c or cache(), seqs=s or seqs(), d_q=P, d_out=P, q_token_stride=4096, q_head_stride=128, out_token_stride=4096,
                            out_head_stride=128, type=0, q_heads=32, scale=0.1, causal=1, d_status=P, d_workspace=P, workspace_bytes=1 << 30)
    for n, v in kw.items():
        setattr(p, n, v)
    return p


def select(c=None, s=None, **kw):
    p = _lib.KvSelectParams(c or cache(), s or seqs(), P, 4096, 128, 0, 32, 3, 1, 1, 1, P, P, 1 << 30, P)
    for n, v in kw.items():
        setattr(p, n, v)
    return p


def evict(c=None, s=None, **kw):
    p = _lib.KvEvictParams(cache=c or cache(), to=cache(), seqs=s or seqs(), d_to_table=P, to_table_stride=4, d_weights=P, weights_seq_stride=512,
                           weights_head_stride=64, d_new_weights=P, new_weights_seq_stride=512, new_weights_head_stride=64, d_kept=P, d_new_lens=P,
                           to_table_width=4, weights_width=64, new_weights_width=64, budget=40, first=1, recent=4, d_status=P)
    for n, v in kw.items():
        setattr(p, n, v)
    return p


CACHES = [dict(d_pages=None), dict(d_pages=P + 8), dict(tokens=0), dict(tokens=8), dict(tokens=24), dict(tokens=272), dict(dim=0), dict(dim=8), dict(dim=100),
          dict(dim=272), dict(heads=0), dict(heads=2000), dict(n_pages=0), dict(n_pages=1 << 31), dict(page_stride=34928), dict(page_stride=34952)]
SEQS = [dict(d_lens=None), dict(d_table=None), dict(n_seqs=0), dict(n_seqs=65536), dict(table_width=0), dict(table_stride=3), dict(n_tokens=3),
        dict(n_tokens=(1 << 24) + 2), dict(table_width=1 << 24, table_stride=1 << 24)]
OPS = {"flh_kv_store": store, "flh_kv_attend": attend, "flh_kv_select": select, "flh_kv_evict": evict}


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("bad", CACHES, ids=str)
def test_caches(lib, op, bad):
    assert getattr(lib, op)(C.byref(OPS[op](c=cache(**bad))), None) == E_ARG
    assert lib.flh_last_error()


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("bad", SEQS, ids=str)
def test_sequences(lib, op, bad):
    assert getattr(lib, op)(C.byref(OPS[op](s=seqs(**bad))), None) == E_ARG
    assert getattr(lib, op)(C.byref(OPS[op](d_status=None)), None) == E_ARG
    assert getattr(lib, op)(None, None) == E_ARG


WIDE = dict(table_width=400, table_stride=400)
CALLS = [("flh_kv_store", dict(type=3)), ("flh_kv_store", dict(d_k=None)), ("flh_kv_store", dict(d_v=None)), ("flh_kv_store", dict(d_k=P + 1)),
         ("flh_kv_attend", dict(type=2)), ("flh_kv_attend", dict(d_q=None)), ("flh_kv_attend", dict(d_out=None)), ("flh_kv_attend", dict(d_q=P + 1)),
         ("flh_kv_attend", dict(q_heads=0)), ("flh_kv_attend", dict(q_heads=33)), ("flh_kv_attend", dict(s=seqs(**WIDE), d_workspace=None)), ("flh_kv_attend", dict(s=seqs(**WIDE), workspace_bytes=64)),
         ("flh_kv_attend", dict(s=seqs(**WIDE), d_workspace=P + 4)), ("flh_kv_attend", dict(d_selected=P)), ("flh_kv_attend", dict(d_selected=P, n_selected=1 << 23)),
         ("flh_kv_attend", dict(d_selected=P, n_selected=2, d_weights=P, weights_width=64)), ("flh_kv_attend", dict(d_weights_in=P)), ("flh_kv_attend", dict(d_weights=P)),
         ("flh_kv_select", dict(type=2)), ("flh_kv_select", dict(d_q=None)), ("flh_kv_select", dict(d_out=None)), ("flh_kv_select", dict(q_heads=9)), ("flh_kv_select", dict(count=0)),
         ("flh_kv_select", dict(first=3)), ("flh_kv_select", dict(last=0xffffffff)), ("flh_kv_select", dict(d_workspace=None)), ("flh_kv_select", dict(workspace_bytes=100)),
         ("flh_kv_evict", dict(to=cache(heads=4))), ("flh_kv_evict", dict(to=cache(dim=64))), ("flh_kv_evict", dict(to=cache(tokens=20))), ("flh_kv_evict", dict(budget=0)),
         ("flh_kv_evict", dict(budget=(1 << 30) + 1)), ("flh_kv_evict", dict(recent=40)), ("flh_kv_evict", dict(to_table_width=2)), ("flh_kv_evict", dict(to_table_stride=3)),
         ("flh_kv_evict", dict(weights_width=0)), ("flh_kv_evict", dict(new_weights_width=39)), ("flh_kv_evict", dict(d_weights=None)), ("flh_kv_evict", dict(d_kept=None)),
         ("flh_kv_evict", dict(d_new_weights=None)), ("flh_kv_evict", dict(d_new_lens=None)), ("flh_kv_evict", dict(d_to_table=None))]


def call_id(call):
    op, fields = call
    return op + " " + ", ".join(f"{k}={v if isinstance(v, (int, float)) else type(v).__name__}" for k, v in fields.items())


@pytest.mark.parametrize("call", CALLS, ids=call_id)
def test_calls(lib, call):
    op, bad = call
    assert getattr(lib, op)(C.byref(OPS[op](**bad)), None) == E_ARG


def test_sizes(lib):
    assert kv.page_bytes(16, 8, 128) == 34944 and kv.page_bytes(16, 1, 16) == 640
    assert lib.flh_kv_page_bytes(256, 1024, 256) == 2 * 1024 * 256 * 256 + 2 * 1024 * 256 + 8 * 1024
    assert lib.flh_kv_attend_workspace_bytes(None) == E_ARG
    assert lib.flh_kv_attend_workspace_bytes(C.byref(attend(s=seqs(n_seqs=0)))) == E_ARG
    assert lib.flh_kv_attend_workspace_bytes(C.byref(attend(q_heads=7))) == E_ARG
    many = attend(c=cache(heads=1024), s=seqs(n_tokens=1 << 24, n_seqs=1), q_heads=1024)
    assert lib.flh_kv_attend(C.byref(many), None) == E_ARG                       # more rows than a launch can number
    assert lib.flh_kv_select(C.byref(select(s=seqs(n_tokens=65536))), None) == E_ARG
    assert lib.flh_kv_select(C.byref(select(c=cache(heads=1024, page_stride=1 << 24), s=seqs(n_tokens=65534), q_heads=1024)), None) == E_ARG
    assert lib.flh_kv_evict(C.byref(evict(c=cache(heads=1024, page_stride=1 << 24), to=cache(heads=1024, page_stride=1 << 24), s=seqs(n_seqs=65535, n_tokens=0))), None) == E_ARG


@pytest.mark.skipif(torch.cuda.is_available(), reason="the refusals below are those of a machine without a GPU")
def test_no_gpu(lib):
    pool = kv.PageCache(torch.zeros(2, kv.page_bytes(16, 1, 16), dtype=torch.uint8), 16, 1, 16)
    k = torch.zeros(2, 1, 16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="no CPU path"):
        kv.store(pool, k, k, i.view(2, 1), i, i)
    if "NCCL_FUSELINK_DEVICE" not in os.environ:
        assert lib.flh_kv_store(C.byref(store()), None) == -3                    # a sound call, and nothing to run it on


def test_wrapper_refusals():
    need = kv.page_bytes(16, 2, 32)
    zeros = lambda *s, d=torch.uint8: torch.zeros(*s, dtype=d)
    for t in (zeros(2, need - 1), zeros(2, need, d=torch.int8), zeros(2 * need), zeros(2, need + 8)[:, 8:], zeros(0, need), zeros(need, 2).t(), zeros(2, need + 8)):
        with pytest.raises(ValueError):
            kv.PageCache(t, 16, 2, 32)
    for tokens, heads, dim in ((8, 2, 32), (272, 2, 32), (16, 0, 32), (16, 2, 24), (16, 2, 512)):
        with pytest.raises(ValueError):
            kv.PageCache(zeros(2, 1 << 20), tokens, heads, dim)
    c = kv.PageCache(zeros(2, need), 16, 2, 32)
    k, i = zeros(2, 2, 32, d=torch.bfloat16), zeros(2, d=torch.int32)
    w = zeros(2, 2, 8, d=torch.float32)
    q = zeros(2, 4, 32, d=torch.float16)
    t = i.view(2, 1)
    bad = [lambda: kv.store(c, k, k.half(), t, i, i), lambda: kv.store(c, k[:, :1], k[:, :1], t, i, i), lambda: kv.store(c, k.double(), k.double(), t, i, i),
           lambda: kv.store(c, k.transpose(1, 2), k.transpose(1, 2), t, i, i), lambda: kv.attend(c, q.float(), t, i, i), lambda: kv.attend(c, q[:, :3], t, i, i),
           lambda: kv.attend(c, q[:, :, :16], t, i, i), lambda: kv.select_pages(c, q, t, i, 2, i, first=2, last=1), lambda: kv.select_pages(c, q, t, i, 0, i),
           lambda: kv.evict(c, t, i, w, 0, c, t, i), lambda: kv.evict(c, t, i, w, 4, c, t, i, first=3, recent=2)]
    for call in bad:
        with pytest.raises(ValueError):
            call()


def apart(**kw):
    """An eviction whose arrays are all memory of their own: a sound call but for `kw`."""
    at = {n: (i + 2) << 32 for i, n in enumerate(("d_to_table", "d_weights", "d_new_weights", "d_kept", "d_new_lens", "d_status"))}
    return evict(**{"to": cache(d_pages=1 << 40), "s": seqs(d_lens=1 << 41, d_table=1 << 42), **at, **kw})


@pytest.mark.parametrize("bad", [fields for op, fields in CALLS if op == "flh_kv_evict"], ids=lambda f: call_id(("flh_kv_evict", f)))
def test_evictions_apart(lib, bad):
    assert lib.flh_kv_evict(C.byref(apart(**bad)), None) == E_ARG
    assert b"overlap" not in lib.flh_last_error()


@pytest.mark.parametrize("shift", [-4, 0, 4])
def test_evict_lengths_in_place(lib, shift):
    """The new lengths of 2 sequences written over what the call's other workgroups may still read."""
    assert lib.flh_kv_evict(C.byref(apart(d_new_lens=(1 << 41) + shift)), None) == E_ARG
    assert b"overlap" in lib.flh_last_error()


def test_evict_onto_the_pages_that_are_read(lib):
    assert lib.flh_kv_evict(C.byref(apart(d_to_table=1 << 42, to=cache())), None) == E_ARG
    assert b"new pages are those" in lib.flh_last_error()


@pytest.mark.parametrize("width", [1 << 31, (1 << 32) - 1024, (1 << 32) - 1])
def test_widths_past_31_bits(lib, width):
    """Rows that a workgroup walks to their end, by strides that would wrap around."""
    for op, p in (("flh_kv_select", select(count=width)), ("flh_kv_attend", attend(d_weights=P, weights_width=width)),
                  ("flh_kv_evict", apart(weights_width=width)), ("flh_kv_evict", apart(new_weights_width=width))):
        assert getattr(lib, op)(C.byref(p), None) == E_ARG


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 3e38])
def test_scales_that_are_not_finite(lib, scale):
    assert lib.flh_kv_attend(C.byref(attend(scale=scale)), None) == E_ARG
    assert b"scale" in lib.flh_last_error()


def test_tensors_that_require_a_gradient():
    need = kv.page_bytes(16, 2, 32)
    c = kv.PageCache(torch.zeros(2, need, dtype=torch.uint8), 16, 2, 32)
    i = torch.zeros(2, dtype=torch.int32)
    t = i.view(2, 1)
    k, q, w = torch.zeros(2, 2, 32), torch.zeros(2, 4, 32, dtype=torch.float16), torch.zeros(2, 2, 32)
    g = lambda x: x.clone().requires_grad_()
    calls = [lambda: kv.store(c, g(k), k, t, i, i), lambda: kv.store(c, k, g(k), t, i, i), lambda: kv.attend(c, g(q), t, i, i), lambda: kv.attend(c, g(q) * 2, t, i, i),
             lambda: kv.attend(c, q, t, i, i, out=g(q)), lambda: kv.attend(c, q, t, i, i, weights=g(w)), lambda: kv.attend(c, q, t, i, i, weights=w, weights_in=g(w)),
             lambda: kv.attend(c, q, t, i, i, lse=g(w[:, :, 0])), lambda: kv.evict(c, t, i, g(w), 16, c, t, i), lambda: kv.evict(c, t, i, w, 16, c, t, i, new_weights=g(w))]
    for call in calls:
        with pytest.raises(ValueError, match="no gradient"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="no CPU path"):     # what comes next here
            call()
