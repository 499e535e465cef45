"""The operators on KV pages held in 8 bits, as cases to measure: their plain forms in elementary torch operations
and the calls a user makes of ``fuselink_amd.kv`` for the same work.

A page record holds T tokens of H key-value heads of D dimensions (all offsets in bytes):

    K codes  e4m3  [H][T][D]     at 0
    V codes  e4m3  [H][T][D]     at H T D
    low      int8  [H][D]        at 2 H T D            floor(smallest K code / 4) over the held tokens
    high     int8  [H][D]        at 2 H T D + H D      ceil(largest K code / 4)
    scales   f32   [H][2]        at 2 H T D + 2 H D    powers of two, of K and of V; value = code * scale
    (rounded up to a multiple of 128)
"""
import math
import random

import torch

own = False

F8 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEV = "cuda"


# ---- the cases ------------------------------------------------------------------------------------------------------
def listed():
    page = dict(T=16, H=8, D=128)      # the paged transfer workload's pages: 16 tokens x 8 heads x 128 dims
    return [
        # prompts of a batch enter the cache on the prefill side: as many tokens as the transfer workload moves, ragged
        dict(name="store_prompts", op="store", B=16, n=4096, ragged=1, held=0, dtype="bf16", **page),
        # one decode step of a batch: one token for each sequence, in the middle of a page
        dict(name="store_token", op="store", B=64, n=1, ragged=0, held=1001, dtype="bf16", **page),
        # the first steps of a single conversation: nothing but latency
        dict(name="attend_first", op="attend", B=1, n=1, ragged=0, len=201, G=4, weights=0, dtype="bf16", **page),
        # an ordinary decode step: a batch of ragged lengths, grouped heads
        dict(name="attend_batch", op="attend", B=32, n=1, ragged=1, len=4096, G=8, weights=0, dtype="bf16", **page),
        # every query head with a cache of its own, pages of 32 tokens, batch 8
        dict(name="attend_ungrouped", op="attend", B=8, n=1, ragged=1, len=4096, G=1, weights=0, dtype="fp16", T=32, H=40, D=128),
        # long documents: the cache passes 4 GiB
        dict(name="attend_long", op="attend", B=16, n=1, ragged=0, len=131072, G=8, weights=0, dtype="bf16", **page),
        # the rest of a prompt against what is cached already: many query tokens for each sequence, causal
        dict(name="attend_chunk", op="attend", B=4, n=1024, ragged=1, len=16384, G=4, weights=0, dtype="bf16", **page),
        # a decode step that keeps account of what was attended to, for the eviction
        dict(name="attend_weights", op="attend", B=16, n=1, ragged=1, len=8192, G=8, weights=1, dtype="bf16", **page),
        # decode steps that read 64 pages of each long sequence instead of all of them
        dict(name="sparse_batch", op="sparse", B=16, n=1, ragged=1, len=32768, G=8, count=64, dtype="bf16", **page),
        # the longest contexts, a small batch
        dict(name="sparse_long", op="sparse", B=4, n=1, ragged=0, len=262144, G=4, count=128, dtype="fp16", **page),
        # a batch of sequences cut back to a quarter of their tokens
        dict(name="evict_batch", op="evict", B=16, ragged=1, len=8192, budget=2048, first=4, recent=256, **page),
        # one short conversation that has just passed its budget
        dict(name="evict_one", op="evict", B=1, ragged=0, len=1040, budget=1024, first=4, recent=64, **page),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        c = dict(op=rng.choice(["store", "attend", "attend", "sparse", "evict"]), B=_log(rng, 1, 64), ragged=rng.randint(0, 1),
                 T=rng.choice([16, 16, 32, 48, 64, 128]), H=rng.choice([1, 2, 3, 5, 8, 8, 12, 16, 40]), D=rng.choice([64, 80, 96, 128, 128, 256]))
        if c["op"] == "store":
            c.update(n=_log(rng, 1, 4096), held=rng.choice([0, 0, 1]) * _log(rng, 1, 2000), dtype=rng.choice(["bf16", "fp16", "fp32"]))
            size = c["B"] * (c["n"] + c["held"])
        elif c["op"] == "attend":
            c.update(n=rng.choice([1, 1, 1, _log(rng, 2, 1024)]), G=rng.choice([1, 2, 4, 7, 8, 16]), weights=rng.choice([0, 0, 1]),
                     dtype=rng.choice(["bf16", "fp16"]), len=_log(rng, 1, 131072))
            size = c["B"] * c["len"] * max(1, c["n"] * c["G"] // 16)
        elif c["op"] == "sparse":
            c.update(n=rng.choice([1, 1, _log(rng, 2, 8)]), G=rng.choice([1, 2, 4, 7, 8, 16]), count=_log(rng, 4, 256),
                     dtype=rng.choice(["bf16", "fp16"]), len=_log(rng, 1, 262144))
            size = c["B"] * (c["len"] + c["n"] * c["count"] * c["T"])
        else:
            c.update(len=_log(rng, 1, 32768))
            c.update(budget=max(8, int(c["len"] * rng.uniform(0.1, 1.2))), first=rng.randint(0, 4), recent=rng.randint(0, 4))
            size = c["B"] * c["len"]
        if size * c["H"] * c["D"] <= 2 ** 29 and c.get("n", 1) <= c.get("len", 1 << 30):
            return c


def _lens(case, seed):
    """Tokens in every sequence; the seed orders them, the sum belongs to the case."""
    full, B = case.get("len", case.get("n")), case["B"]
    lens = [max(1, full - (full * 3 // 4) * i // B) if case["ragged"] else full for i in range(B)]
    random.Random(seed).shuffle(lens)
    return lens


def _news(case, lens):
    """Query tokens of every sequence."""
    return [min(case["n"], x) if not case["ragged"] else max(1, min(x, case["n"] - (i % 4) * (case["n"] // 8))) for i, x in enumerate(lens)]


def work(case):
    T, H, D = case["T"], case["H"], case["D"]
    lens = _lens(case, 0)
    if case["op"] == "store":
        n, e = sum(lens), 4 if case["dtype"] == "fp32" else 2
        pages = sum((x + T - 1) // T for x in lens)
        return {"bytes": n * H * D * 2 * (e + 1) + pages * H * (2 * D + 8), "flops": n * H * D * 4}
    if case["op"] == "evict":
        kept = sum(min(x, case["budget"]) for x in lens)
        return {"bytes": sum(lens) * H * 4 + kept * H * (4 * D + 8), "flops": kept * H * D * 4}
    if case["op"] == "attend":
        news = _news(case, lens)
        total = sum(lens)
        seen = sum(n * x - n * (n - 1) // 2 for n, x in zip(news, lens))
        rows = sum(news) * H * case["G"]
        b = total * H * 2 * D + total // T * H * 8 + rows * D * 4 + (total * H * 8 if case["weights"] else 0)
        return {"bytes": b, "flops": seen * H * case["G"] * D * 4}
    news = _news(case, lens)
    pages = sum((x + T - 1) // T for x in lens)
    read = sum(n * min(x, case["count"] * T) for n, x in zip(news, lens))
    b = pages * H * (2 * D + 4) + read * H * 2 * D + sum(news) * H * (case["G"] * D * 4 + case["count"] * 4)
    return {"bytes": b, "flops": (sum(n * ((x + T - 1) // T) for n, x in zip(news, lens)) * 2 + read * 4) * H * case["G"] * D}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def page_bytes(T, H, D):
    return (2 * H * T * D + 2 * H * D + 8 * H + 127) // 128 * 128


def _views(pages, T, H, D):
    """K codes, V codes, low, high and scales of a pool of records, as views."""
    a, n = H * T * D, pages.shape[0]
    return (pages[:, :a].view(F8).view(n, H, T, D), pages[:, a:2 * a].view(F8).view(n, H, T, D),
            pages[:, 2 * a:2 * a + H * D].view(torch.int8).view(n, H, D), pages[:, 2 * a + H * D:2 * a + 2 * H * D].view(torch.int8).view(n, H, D),
            pages[:, 2 * a + 2 * H * D:2 * a + 2 * H * D + 8 * H].view(torch.float32).view(n, H, 2))


def _pow2(e):
    """2^e, exactly, in 32 bits."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _scale(amax):
    """The smallest power of two s with amax <= 448 s."""
    f, x = torch.frexp(amax)
    return torch.where(amax > 0, _pow2(torch.where(f <= 0.875, x - 9, x - 8).clamp(min=-126)), 0)


def _pack(values, held, least):
    """Values [..., T, D] of blocks of tokens, the slots that hold one [..., T], and the least scale [...] -> codes, scales."""
    ok = torch.isfinite(values) & held[..., None]
    s = torch.maximum(_scale(torch.where(ok, values.abs(), 0).amax((-1, -2))), least)
    inv = torch.where(s > 0, 1 / torch.where(s > 0, s, 1), 0)[..., None, None]
    codes = torch.where(ok, values * inv, torch.where(held[..., None], math.nan, 0.0)).to(F8)
    return codes, s


def _bounds(codes, held):
    """floor / ceil of a quarter of the smallest and largest code of every channel: codes [..., T, D] -> two of [..., D]."""
    c = codes.float()
    ok = torch.isfinite(c) & held[..., None]
    any_ = ok.any(-2)
    lo = torch.where(any_, torch.floor(torch.where(ok, c, 1e9).amin(-2) / 4), 0)
    hi = torch.where(any_, torch.ceil(torch.where(ok, c, -1e9).amax(-2) / 4), 0)
    return lo.to(torch.int8), hi.to(torch.int8)


def _gains(g, H, D):
    """Channels differ in size, a few by much, in keys more than in values."""
    k = torch.exp(0.3 * torch.randn(H, D, generator=g, device=DEV))
    k[:, torch.randperm(D, generator=g, device=DEV)[:2]] *= 5
    return k, torch.exp(0.2 * torch.randn(H, D, generator=g, device=DEV)), torch.randn(H, D, generator=g, device=DEV)


def _tokens(g, n, H, D, gains, first):
    k = torch.randn(n, H, D, generator=g, device=DEV) * gains[0]
    v = torch.randn(n, H, D, generator=g, device=DEV) * gains[1]
    if first:                  # the first token draws attention and has little to say
        k[0] = gains[2] * 3
        v[0] *= 0.05
    return k, v


def _fill(g, T, H, D, lens, spare):
    """A pool of records that holds len tokens of every sequence, in pages of a random order."""
    counts = [(x + T - 1) // T + spare for x in lens]
    n_pages = sum(counts) + 3
    pages = torch.zeros(n_pages, page_bytes(T, H, D), dtype=torch.uint8, device=DEV)
    order = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(lens), max(max(counts), 1)), -1, dtype=torch.int32, device=DEV)
    kc, vc, lo, hi, sc = _views(pages, T, H, D)
    gains, at = _gains(g, H, D), 0
    step = max(T, (1 << 25) // (H * D) // T * T)
    for b, x in enumerate(lens):
        table[b, :counts[b]] = order[at:at + counts[b]]
        for t0 in range(0, x, step):
            m = min(step, x - t0)
            k, v = _tokens(g, m, H, D, gains, t0 == 0)
            p = (m + T - 1) // T
            held = (torch.arange(p * T, device=DEV) < m).view(p, 1, T)
            ids = table[b, t0 // T:t0 // T + p].long()
            for side, (val, codes) in enumerate(((k, kc), (v, vc))):
                val = torch.nn.functional.pad(val, (0, 0, 0, 0, 0, p * T - m)).view(p, T, H, D).transpose(1, 2)
                c, s = _pack(val, held, torch.zeros(p, H, device=DEV))
                codes.view(torch.uint8)[ids] = c.view(torch.uint8)
                sc[ids, :, side] = s
                if side == 0:
                    lo[ids], hi[ids] = _bounds(c, held)
        at += counts[b]
    return pages, table, gains


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    T, H, D = case["T"], case["H"], case["D"]
    lens = _lens(case, seed)
    st = dict(case=case, status=torch.zeros(1, dtype=torch.int32, device=DEV))
    if case["op"] == "store":
        news, held = lens, [case["held"]] * case["B"]
        st["pages"], st["table"], gains = _fill(g, T, H, D, held, (max(news) + T - 1) // T + 1)
        parts = [_tokens(g, n, H, D, gains, case["held"] == 0) for n in news]
        st["k"], st["v"] = (torch.cat([p[i] for p in parts]).to(TYPES[case["dtype"]]) for i in (0, 1))
        st["lens"] = torch.tensor(held, dtype=torch.int32, device=DEV)
    elif case["op"] == "evict":
        news = [1] * case["B"]
        st["pages"], st["table"], _ = _fill(g, T, H, D, lens, 0)
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        width = (max(lens) + 63) // 64 * 64
        w = torch.exp(2 * torch.randn(case["B"], H, width, generator=g, device=DEV))
        st["weights"] = torch.where(torch.rand(w.shape, generator=g, device=DEV) < 0.05, 0, w)      # never attended to
        per = (case["budget"] + T - 1) // T
        n_new = case["B"] * per
        st["new_pages"] = torch.zeros(n_new, page_bytes(T, H, D), dtype=torch.uint8, device=DEV)
        st["new_table"] = torch.randperm(n_new, generator=g, device=DEV).to(torch.int32).view(case["B"], per)
    else:
        news = _news(case, lens)
        st["pages"], st["table"], gains = _fill(g, T, H, D, lens, 0)
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        q = torch.randn(sum(news), H, case["G"], D, generator=g, device=DEV) + 0.5 * gains[2][:, None]
        st["q"] = q.reshape(sum(news), H * case["G"], D).to(TYPES[case["dtype"]])
        if case.get("weights"):
            st["weights"] = torch.rand(case["B"], H, (max(lens) + 63) // 64 * 64, generator=g, device=DEV)
            st["weights_out"] = torch.empty_like(st["weights"])
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    st["starts"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
    # a program's scheduler knows on the host how long its sequences are
    st["host"] = dict(lens=lens, news=news, starts=starts)
    if case["op"] in ("store", "evict"):       # what the call writes, as views of the pool
        k, v, lo, hi, sc = _views(st["pages" if case["op"] == "store" else "new_pages"], T, H, D)
        st["records"] = dict(k=k, v=v, low=lo, high=hi, scales=sc)
    if own:
        from fuselink_amd import kv
        st["cache"] = kv.PageCache(st["pages"], tokens=T, heads=H, dim=D)
        if case["op"] == "evict":
            st["new_cache"] = kv.PageCache(st["new_pages"], tokens=T, heads=H, dim=D)
    return st


# ---- the framework's calls ------------------------------------------------------------------------------------------
def _own(st):
    from fuselink_amd import kv
    case = st["case"]
    starts = st["starts"]
    if case["op"] == "store":
        kv.store(st["cache"], st["k"], st["v"], st["table"], st["lens"], st["status"], starts=starts)
        return st["records"]
    if case["op"] == "evict":
        kept, weights, lens = kv.evict(st["cache"], st["table"], st["lens"], st["weights"], case["budget"], st["new_cache"], st["new_table"], st["status"],
                                       first=case["first"], recent=case["recent"])
        return dict(st["records"], kept=kept, weights=weights, lens=lens)
    if case["op"] == "sparse":
        sel = kv.select_pages(st["cache"], st["q"], st["table"], st["lens"], case["count"], st["status"], starts=starts, first=1, last=2)
        return dict(selected=sel, out=kv.attend(st["cache"], st["q"], st["table"], st["lens"], st["status"], starts=starts, selected=sel))
    if case["weights"]:
        out = kv.attend(st["cache"], st["q"], st["table"], st["lens"], st["status"], starts=starts, weights=st["weights_out"], weights_in=st["weights"])
        return dict(out=out, weights=st["weights_out"])
    return kv.attend(st["cache"], st["q"], st["table"], st["lens"], st["status"], starts=starts)


# ---- the plain forms ------------------------------------------------------------------------------------------------
def _values(st, b, n):
    """K and V of the first n tokens of sequence b, [H, n, D] in 32 bits."""
    case = st["case"]
    T, H, D = case["T"], case["H"], case["D"]
    kc, vc, _, _, sc = _views(st["pages"], T, H, D)
    ids = st["table"][b, :(n + T - 1) // T].long()
    return tuple((c.view(torch.uint8)[ids].view(F8).float() * sc[ids, :, i, None, None]).transpose(0, 1).reshape(H, -1, D)[:, :n] for i, c in enumerate((kc, vc)))


def _softmax_out(q, k, v, seen, c):
    """q [H, R, D] over k, v [H, n, D]; seen [R, n] or [H, R, n]: outputs [H, R, D] and probabilities [H, R, n]."""
    s = torch.where(seen, torch.matmul(q, k.transpose(1, 2).contiguous()) * c, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    return torch.matmul(p, v), p


def _rows(q, H, G):
    """Query tokens [n, H G, D] -> rows of every key-value head [H, n G, D]."""
    n, _, D = q.shape
    return q.view(n, H, G, D).transpose(0, 1).reshape(H, n * G, D)


def _plain_attend(st):
    case, host = st["case"], st["host"]
    H, G, D = case["H"], case["G"], case["D"]
    out = torch.empty_like(st["q"])
    weights = st["weights"].clone() if case["weights"] else None
    for b, (n, x) in enumerate(zip(host["news"], host["lens"])):
        lo, hi = host["starts"][b], host["starts"][b + 1]
        k, v = _values(st, b, x)
        per = max(1, (1 << 28) // max(1, H * G * x))       # query tokens at a time: scores of up to 1 GiB
        for t in range(0, n, per):
            m = min(per, n - t)
            pos = torch.arange(x - n + t, x - n + t + m, device=DEV).repeat_interleave(G)
            o, p = _softmax_out(_rows(st["q"][lo + t:lo + t + m].float(), H, G), k, v, torch.arange(x, device=DEV) <= pos[:, None], 1 / math.sqrt(D))
            out[lo + t:lo + t + m] = o.view(H, m, G, D).transpose(0, 1).reshape(m, H * G, D).to(out.dtype)
            if weights is not None:
                weights[b, :, :x] += p.sum(1)
    return out if weights is None else dict(out=out, weights=weights)


def _eighth(q):
    """Eight-bit whole numbers of every query head and their power-of-two step."""
    a = q.abs().amax(-1, keepdim=True)
    f, x = torch.frexp(a)
    s = torch.where(a > 0, _pow2(torch.where(f <= 0.9921875, x - 7, x - 6).clamp(min=-126)), 1)
    return torch.round(q / s), torch.where(a > 0, s, 0)


def _best(score, count, first, last):
    """Indices, ascending, of the `count` best of score [..., n]; the first and last ones come before all; -1 behind them."""
    n = score.shape[-1]
    score = score.clone()
    score[..., :first] = math.inf
    score[..., max(0, n - last):] = math.inf
    k = min(count, n)
    idx = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :k].sort(-1).values.to(torch.int32)
    return torch.nn.functional.pad(idx, (0, count - k), value=-1)


def _plain_sparse(st):
    case, host = st["case"], st["host"]
    T, H, G, D, count = case["T"], case["H"], case["G"], case["D"], case["count"]
    kc, vc, low, high, sc = _views(st["pages"], T, H, D)
    out = torch.empty_like(st["q"])
    sel = torch.empty(out.shape[0], H, count, dtype=torch.int32, device=DEV)
    heads = torch.arange(H, device=DEV)[:, None]
    for b, (n, x) in enumerate(zip(host["news"], host["lens"])):
        for t in range(n):
            row, seen = host["starts"][b] + t, x - n + t + 1
            ids = st["table"][b, :(seen + T - 1) // T].long()
            lo, hi = low[ids].transpose(0, 1).float(), high[ids].transpose(0, 1).float()                    # [H, pages, D]
            q8, step = _eighth(st["q"][row].view(H, G, D).float())
            whole = torch.matmul(hi, q8.clamp(min=0).transpose(1, 2).contiguous()) + torch.matmul(lo, q8.clamp(max=0).transpose(1, 2).contiguous())
            score = (whole * step.transpose(1, 2)).amax(-1) * sc[ids, :, 0].transpose(0, 1)
            sel[row] = _best(score, count, 1, 2)
            mine = sel[row].long()
            pg = ids[mine.clamp(min=0)]                                                                     # [H, count]
            pos = mine[..., None] * T + torch.arange(T, device=DEV)
            ok = ((mine[..., None] >= 0) & (pos < seen)).view(H, 1, -1)
            k, v = ((c.view(torch.uint8)[pg, heads].view(F8).float() * sc[pg, heads, i][..., None, None]).view(H, -1, D) for i, c in enumerate((kc, vc)))
            o, _ = _softmax_out(_rows(st["q"][row:row + 1].float(), H, G), k, v, ok, 1 / math.sqrt(D))
            out[row] = o.view(H * G, D).to(out.dtype)
    return dict(selected=sel, out=out)


def _plain_store(st):
    case, host = st["case"], st["host"]
    T, H, D = case["T"], case["H"], case["D"]
    kc, vc, lo, hi, sc = _views(st["pages"], T, H, D)
    held = case["held"]
    for b, n in enumerate(host["news"]):
        first, end = held // T, (held + n + T - 1) // T
        ids = st["table"][b, first:end].long()
        p, skip = end - first, held - first * T
        slot = torch.arange(p * T, device=DEV).view(p, 1, T)
        old, now = slot < skip, slot < skip + n
        for side, (src, codes) in enumerate(((st["k"], kc), (st["v"], vc))):
            new = src[host["starts"][b]:host["starts"][b] + n].float()
            new = torch.nn.functional.pad(new, (0, 0, 0, 0, skip, p * T - skip - n)).view(p, T, H, D).transpose(1, 2)
            was = sc[ids, :, side] * old.any(-1)
            val = torch.where(old[..., None], codes.view(torch.uint8)[ids].view(F8).float() * was[..., None, None], new)
            c, s = _pack(val, now, was)
            codes.view(torch.uint8)[ids] = c.view(torch.uint8)
            sc[ids, :, side] = s
            if side == 0:
                lo[ids], hi[ids] = _bounds(c, now)
    return st["records"]


def _plain_evict(st):
    case, host = st["case"], st["host"]
    T, H, D, budget = case["T"], case["H"], case["D"], case["budget"]
    B, per = st["new_table"].shape
    kc, vc, lo, hi, sc = _views(st["new_pages"], T, H, D)
    kept = torch.full((B, H, budget), -1, dtype=torch.int32, device=DEV)
    weights = torch.zeros(B, H, budget, device=DEV)
    for b, x in enumerate(host["lens"]):
        m = min(x, budget)
        if x <= budget:
            idx = torch.arange(x, device=DEV, dtype=torch.int32).expand(H, x)
        else:
            idx = _best(st["weights"][b, :, :x], budget, case["first"], case["recent"])
        kept[b, :, :m] = idx
        weights[b, :, :m] = torch.gather(st["weights"][b], 1, idx.long())
        p = (m + T - 1) // T
        ids = st["new_table"][b, :p].long()
        held = (torch.arange(p * T, device=DEV) < m).view(p, 1, T)
        for side, (val, codes) in enumerate(zip(_values(st, b, x), (kc, vc))):
            val = torch.gather(val, 1, idx.long()[..., None].expand(H, m, D))
            val = torch.nn.functional.pad(val, (0, 0, 0, p * T - m)).view(H, p, T, D).transpose(0, 1)
            c, s = _pack(val, held, torch.zeros(p, H, device=DEV))
            codes.view(torch.uint8)[ids] = c.view(torch.uint8)
            sc[ids, :, side] = s
            if side == 0:
                lo[ids], hi[ids] = _bounds(c, held)
    return dict(st["records"], kept=kept, weights=weights, lens=st["lens"].clamp(max=budget))


def run(state):
    if own:
        return _own(state)
    return {"store": _plain_store, "attend": _plain_attend, "sparse": _plain_sparse, "evict": _plain_evict}[state["case"]["op"]](state)


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def _power(e):
    """2^e, exactly, in 64 bits."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _e4m3(b):
    """The numbers that bytes stand for: sign, 4 bits of exponent (bias 7), 3 of mantissa; 0x7f is no number."""
    n = torch.arange(256, dtype=torch.float64, device=DEV)
    s, e, m = torch.where(n >= 128, -1.0, 1.0), torch.floor(n / 8) % 16, n % 8
    t = s * torch.where(e == 0, m / 512, (1 + m / 8) * _power(e - 7))
    t[127] = t[255] = math.nan
    return t[b.long()]


def _nearest(x):
    """The e4m3 number next to x (|x| <= 448), ties to the even one."""
    step = _power(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _least_power(a):
    """The least power of two s with a <= 448 s, by trying its neighbours."""
    e = torch.floor(torch.log2((a / 448).clamp(min=2.0 ** -126)))
    s = _power(e - 1)
    for _ in range(3):
        s = torch.where(a > 448 * s, 2 * s, s)
    return torch.where(a > 0, s.clamp(min=2.0 ** -126), 0.0)


def _bytes64(pages, case, ids, side):
    """Codes [p, H, T, D] and scales [p, H] of records, in 64 bits."""
    T, H, D = case["T"], case["H"], case["D"]
    a = H * T * D
    rec = pages[ids]
    codes = _e4m3(rec[:, side * a:(side + 1) * a]).view(-1, H, T, D)
    off = 2 * a + 2 * H * D
    return codes, rec[:, off:off + 8 * H].contiguous().view(torch.float32).view(-1, H, 2)[..., side].double()


def exact(case, seed):
    st = prepare(case, seed)
    T, H, D = case["T"], case["H"], case["D"]
    lens, news, starts = st["host"]["lens"], st["host"]["news"], st["host"]["starts"]
    if case["op"] == "store":
        ids_all = torch.arange(st["pages"].shape[0], device=DEV)
        res = {}
        for side, name in enumerate("kv"):
            parts = [_bytes64(st["pages"], case, c, side) for c in ids_all.split(512)]
            codes, scales = torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])
            for b, n in enumerate(news):
                at = case["held"]
                for slot in range(at // T, (at + n + T - 1) // T):
                    pg = int(st["host"].setdefault("table", st["table"].tolist())[b][slot])
                    lo, hi = max(at, slot * T), min(at + n, slot * T + T)
                    new = st[name][starts[b] + lo - at:starts[b] + hi - at].double().transpose(0, 1)
                    s0 = scales[pg] if lo > slot * T else torch.zeros_like(scales[pg])
                    s = torch.maximum(s0, _least_power(new.abs().amax((1, 2))))
                    codes[pg, :, :lo - slot * T] = _nearest(codes[pg, :, :lo - slot * T] * torch.where(s > 0, s0 / s, 0.0)[:, None, None])
                    codes[pg, :, lo - slot * T:hi - slot * T] = _nearest(new / torch.where(s > 0, s, 1.0)[:, None, None])
                    codes[pg, :, hi - slot * T:] = 0
                    scales[pg] = s
            res[name], res["s" + name] = codes, scales
        return dict(k=res["k"], v=res["v"], low=None, high=None, scales=torch.stack([res["sk"], res["sv"]], -1))
    if case["op"] == "evict":
        out = {n: torch.zeros(st["new_pages"].shape[0], H, T, D, dtype=torch.float64, device=DEV) for n in "kv"}
        scales = torch.zeros(st["new_pages"].shape[0], H, 2, dtype=torch.float64, device=DEV)
        weights = torch.zeros(case["B"], H, case["budget"], dtype=torch.float64, device=DEV)
        for b, x in enumerate(lens):
            m, w = min(x, case["budget"]), st["weights"][b, :, :x].double()
            if x > m:
                w0 = w.clone()
                w0[:, :case["first"]] = math.inf
                if case["recent"]:
                    w0[:, -case["recent"]:] = math.inf
                order = torch.argsort(-w0, dim=1, stable=True)[:, :m].sort(1).values
            else:
                order = torch.arange(x, device=DEV).repeat(H, 1)
            weights[b, :, :m] = w.gather(1, order)
            ids = st["table"][b, :(x + T - 1) // T].long()
            for side, name in enumerate("kv"):
                codes, s = _bytes64(st["pages"], case, ids, side)
                flat = (codes * s[..., None, None]).permute(1, 0, 2, 3).reshape(H, -1, D)
                for h in range(H):
                    val = flat[h, order[h]]
                    for j, pg in enumerate(st["new_table"][b].tolist()[:(m + T - 1) // T]):
                        blk = val[j * T:(j + 1) * T]
                        sn = _least_power(blk.abs().amax())
                        out[name][pg, h, :blk.shape[0]] = _nearest(blk / torch.where(sn > 0, sn, 1.0))
                        scales[pg, h, side] = sn
        return dict(k=out["k"], v=out["v"], low=None, high=None, scales=scales, kept=None, weights=weights, lens=None)
    G, q, res = case["G"], st["q"].double(), torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    acc = st["weights"].double() if case.get("weights") else None
    if sum(n * x for n, x in zip(news, lens)) * H * G * D > 2 ** 42:
        return None
    for b, (n, x) in enumerate(zip(news, lens)):
        ids = st["table"][b, :(x + T - 1) // T].long()
        for h in range(H):
            (k, ks), (v, vs) = (_head64(st["pages"], case, ids, side, h) for side in (0, 1))
            kk, vv = (k * ks[:, None, None]).view(-1, D)[:x], (v * vs[:, None, None]).view(-1, D)[:x]
            for t in range(0, n, 64):
                mine = q[starts[b] + t:starts[b] + min(n, t + 64), h * G:(h + 1) * G]
                seen = x - n + 1 + torch.arange(t, t + mine.shape[0], device=DEV)
                use = (torch.arange(x, device=DEV) < seen[:, None])
                if case["op"] == "sparse":
                    use = torch.stack([u & _chosen64(st, case, ids, h, mine[i], int(seen[i])).repeat_interleave(T)[:x] for i, u in enumerate(use)])
                s = (mine.reshape(-1, D) @ kk.t().contiguous()).view(-1, G, x) / math.sqrt(D)
                s = s.masked_fill(~use[:, None], -math.inf)
                p = (s - s.amax(-1, keepdim=True)).exp()
                p /= p.sum(-1, keepdim=True)
                res[starts[b] + t:starts[b] + t + mine.shape[0], h * G:(h + 1) * G] = (p.view(-1, x) @ vv).view(-1, G, D)
                if acc is not None:
                    acc[b, h, :x] += p.sum((0, 1))
    if case["op"] == "sparse":
        return dict(selected=None, out=res)
    return res if acc is None else dict(out=res, weights=acc)


def _head64(pages, case, ids, side, h):
    T, H, D = case["T"], case["H"], case["D"]
    a = H * T * D
    off = side * a + h * T * D
    codes = _e4m3(pages[:, off:off + T * D][ids]).view(-1, T, D)
    at = 2 * a + 2 * H * D + 8 * h + 4 * side
    return codes, pages[:, at:at + 4][ids].contiguous().view(torch.float32).view(-1).double()


def _chosen64(st, case, ids, h, q, seen):
    """Truth values over a sequence's pages: those that the bounds of head h make the best for q [G, D]."""
    T, H, D = case["T"], case["H"], case["D"]
    n = (seen + T - 1) // T
    at = 2 * H * T * D + h * D
    lo, hi = (st["pages"][:, at + i * H * D:at + i * H * D + D][ids[:n]].view(torch.int8).double() for i in (0, 1))
    amax = q.abs().amax(-1, keepdim=True)
    step = _power(torch.ceil(torch.log2(amax / 127).clamp(min=-126)))
    step = torch.where(amax <= 127 * step / 2, step / 2, torch.where(amax > 127 * step, 2 * step, step))
    q8 = torch.where(amax > 0, torch.round(q / step), 0.0)
    ks = _head64(st["pages"], case, ids[:n], 0, h)[1]
    score = ((torch.where(q8[:, None] > 0, hi, lo) * q8[:, None]).sum(-1) * step).amax(0) * ks
    score[:1] = math.inf
    score[max(0, n - 2):] = math.inf
    pick = torch.zeros(len(ids), dtype=torch.bool, device=DEV)
    pick[torch.argsort(-score, stable=True)[:case["count"]]] = True
    return pick
