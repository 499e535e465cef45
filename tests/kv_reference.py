"""The operators on KV pages held in 8 bits, from their definitions, in 64 bits on the CPU: plain loops over numpy
arrays, for the tests to compare with.  A cache is a dict of arrays, one entry per page."""
import numpy as np

CODES = np.empty(256)
for _b in range(256):
    _e, _m = (_b >> 3) & 15, _b & 7
    _v = np.nan if (_b & 127) == 127 else (_m * 2.0 ** -9 if _e == 0 else (1 + _m / 8) * 2.0 ** (_e - 7))
    CODES[_b] = -_v if _b & 128 else _v


def page_bytes(T, H, D):
    return -(-(2 * H * T * D + 2 * H * D + 8 * H) // 128) * 128


def unpack(raw, T, H, D):
    """Records (uint8 [n, >= page_bytes]) -> dict of K, V codes as numbers, low, high, scales."""
    n, a = raw.shape[0], H * T * D
    at = 2 * a + 2 * H * D
    return dict(k=CODES[raw[:, :a]].reshape(n, H, T, D), v=CODES[raw[:, a:2 * a]].reshape(n, H, T, D),
                low=raw[:, 2 * a:2 * a + H * D].copy().view(np.int8).reshape(n, H, D),
                high=raw[:, 2 * a + H * D:at].copy().view(np.int8).reshape(n, H, D),
                s=raw[:, at:at + 8 * H].copy().view(np.float32).astype(np.float64).reshape(n, H, 2))


def empty(n, T, H, D):
    return unpack(np.zeros((n, page_bytes(T, H, D)), np.uint8), T, H, D)


def nearest(x):
    """The e4m3 number next to x, ties to the one with the even mantissa; not-finite becomes NaN."""
    x = np.where(np.isfinite(x), x, np.nan)
    _, e = np.frexp(np.abs(np.nan_to_num(x)))
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    return np.round(x / step) * step


def least_power(a, most, floor=-126):
    """The least 2^e >= a / most with e >= floor; 0 for 0."""
    if not a > 0:
        return 0.0
    e = floor
    while a > most * 2.0 ** e:
        e += 1
    return 2.0 ** e


def _amax(x):
    x = np.abs(x[np.isfinite(x)])
    return x.max() if x.size else 0.0


def _set_bounds(c, pg, h, fill):
    for d in range(c["k"].shape[3]):
        col = c["k"][pg, h, :fill, d]
        col = col[~np.isnan(col)]
        c["low"][pg, h, d] = np.floor(col.min() / 4) if col.size else 0
        c["high"][pg, h, d] = np.ceil(col.max() / 4) if col.size else 0


def store(c, k, v, table, lens, starts):
    T, H = c["k"].shape[2], c["k"].shape[1]
    for b in range(len(lens)):
        n, held = starts[b + 1] - starts[b], lens[b]
        for j in range(held // T, -(-(held + n) // T) if n else 0):
            pg, lo, hi = table[b][j], max(held, j * T), min(held + n, (j + 1) * T)
            for h in range(H):
                for side, (name, src) in enumerate((("k", k), ("v", v))):
                    new = src[starts[b] + lo - held:starts[b] + hi - held, h]
                    old = lo - j * T
                    s0 = c["s"][pg, h, side] if old else 0.0
                    s = max(s0, least_power(_amax(new), 448))
                    blk = c[name][pg, h]
                    if old and s != s0:
                        blk[:old] = nearest(blk[:old] * (s0 / s))
                    new = np.where(np.isfinite(new), new, np.nan)
                    blk[old:hi - j * T] = nearest(new / s if s else new * 0)
                    if not old:
                        blk[hi - j * T:] = 0
                    c["s"][pg, h, side] = s
                _set_bounds(c, pg, h, hi - j * T)


def values(c, table_row, h, n):
    """K and V of the first n tokens of a sequence, in 64 bits."""
    T = c["k"].shape[2]
    pages = table_row[:-(-n // T)]
    out = []
    for side, name in enumerate("kv"):
        x = [c[name][p, h] * c["s"][p, h, side] for p in pages]
        out.append(np.concatenate(x)[:n] if x else np.zeros((0, c["k"].shape[3])))
    return out


def attend(c, q, table, lens, starts, scale, causal=True, selected=None, q_bits=None):
    """Outputs, logarithms of sums, attention weights of every key [B][H, len] and the sizes that errors scale with."""
    T, H, D = c["k"].shape[2], c["k"].shape[1], c["k"].shape[3]
    G = q.shape[1] // H
    out, lse = np.zeros(q.shape), np.full(q.shape[:2], -np.inf)
    spread, slack = np.zeros(q.shape), np.zeros(q.shape[:2])       # sum p |v|; error of a score
    weights = [np.zeros((H, x)) for x in lens]
    wslack = [np.zeros((H, x)) for x in lens]
    for b, x in enumerate(lens):
        n = starts[b + 1] - starts[b]
        for h in range(H):
            k, v = values(c, table[b], h, x)
            heads = slice(h * G, (h + 1) * G)
            seen = np.clip(x - n + 1 + np.arange(n), 0, None) if causal else np.full(n, x)
            if selected is None:             # all tokens of the sequence together
                blocks = [(np.arange(n), np.arange(x), np.arange(x)[None] < seen[:, None])]
            else:
                pick = [set(int(j) for j in selected[starts[b] + i, h] if j >= 0) for i in range(n)]
                use = [np.array([j for j in range(seen[i]) if j // T in pick[i]], int) for i in range(n)]
                blocks = [(np.array([i]), u, np.ones((1, len(u)), bool)) for i, u in enumerate(use)]
            for tok, use, vis in blocks:
                tok, vis = tok[vis.any(1)], vis[vis.any(1)]
                if not len(tok):
                    continue
                at, vis, kk, vv = starts[b] + tok, np.repeat(vis, G, 0), k[use], v[use]
                rows, shape = q[at, heads].reshape(-1, D), (len(tok), G)
                s = np.where(vis, rows @ kk.T * scale, -np.inf)
                m = s.max(1, keepdims=True)
                p = np.where(vis, np.exp(s - m), 0)
                tot = p.sum(1, keepdims=True)
                p /= tot
                nan = np.isnan(vv)
                o = p @ np.where(nan, 0, vv)
                o[vis.astype(float) @ nan > 0] = np.nan
                out[at, heads], lse[at, heads] = o.reshape(*shape, D), (m + np.log(tot)).reshape(shape)
                # 32-bit sums of D products, the scaling, and the exponential's argument
                err = (np.abs(rows) @ np.abs(kk).T * abs(scale) * (D + 4) + np.abs(np.where(vis, s, 0)) * 4 + np.abs(m) * 4 + 32) * 2.0 ** -24
                err = np.where(vis, err, 0)
                slack[at, heads] = err.max(1).reshape(shape)
                spread[at, heads] = (p @ np.abs(np.where(nan, 0, vv))).reshape(*shape, D)
                weights[b][h, use] += p.sum(0)
                wslack[b][h, use] += (p * (err + err.max(1, keepdims=True))).sum(0)
    return dict(out=out, lse=lse, weights=weights, spread=spread, slack=slack, wslack=wslack)


def out_tolerance(ref, eps, n_max):
    """How far an output may be off: half a step of its type; each probability rounded to 11 bits (2^-11); twice the error of
    the scores, in the numerator and in the sum; sums of n terms in 32 bits; 16-bit floats below 2^-28 of the largest
    probability are spaced by 2^-38 of it."""
    return np.abs(ref["out"]) * eps / 2 * 1.01 + ref["spread"] * (2.0 ** -11 + 2.2 * ref["slack"][..., None] + (n_max + 64) * 2.0 ** -23) + 1e-30


def eighth(q):
    s = least_power(_amax(q), 127)
    return (np.round(np.where(np.isfinite(q), q, 0.0) / s) if s else q * 0), s


def best(score, count, first, last):
    n = len(score)
    key = [(-np.inf if np.isnan(x) else x) for x in score]
    order = sorted(range(n), key=lambda i: (not (i < first or i >= n - last), np.isnan(score[i]), -key[i], i))
    return sorted(order[:count])


def select(c, q, table, lens, starts, count, first, last, causal=True):
    T, H = c["k"].shape[2], c["k"].shape[1]
    G = q.shape[1] // H
    out = np.full((q.shape[0], H, count), -1, np.int64)
    for b, x in enumerate(lens):
        n = starts[b + 1] - starts[b]
        for i in range(n):
            seen = max(0, x - n + i + 1) if causal else x
            for h in range(H):
                score = []
                for j in range(-(-seen // T)):
                    pg = table[b][j]
                    tops = []
                    for g in range(G):
                        q8, s = eighth(q[starts[b] + i, h * G + g])
                        tops.append(np.where(q8 > 0, c["high"][pg, h], c["low"][pg, h]).astype(np.float64) @ q8 * s)
                    score.append(max(tops) * c["s"][pg, h, 0])
                got = best(score, count, first, last)
                out[starts[b] + i, h, :len(got)] = got
    return out


def evict(c, table, lens, weights, budget, first, recent, to, to_table):
    T, H, D = c["k"].shape[2], c["k"].shape[1], c["k"].shape[3]
    T2 = to["k"].shape[2]
    kept = np.full((len(lens), H, budget), -1, np.int64)
    nw = np.zeros((len(lens), H, budget))
    for b, x in enumerate(lens):
        m = min(x, budget)
        for h in range(H):
            idx = list(range(x)) if x <= budget else best(list(weights[b, h, :x].astype(np.float64)), budget, first, recent)
            kept[b, h, :m] = idx
            nw[b, h, :m] = weights[b, h, idx]
            for side, (name, val) in enumerate(zip("kv", values(c, table[b], h, x))):
                val = val[idx]
                for j in range(-(-m // T2)):
                    pg, blk = to_table[b][j], val[j * T2:(j + 1) * T2]
                    s = least_power(_amax(blk), 448)
                    to[name][pg, h] = 0
                    to[name][pg, h, :len(blk)] = nearest(blk / s if s else blk * 0)
                    to["s"][pg, h, side] = s
                    if side == 0:
                        _set_bounds(to, pg, h, len(blk))
    return kept, nw
