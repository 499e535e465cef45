"""KV pages held in 8 bits: store, attention, the choice of pages and eviction against plain definitions in 64 bits."""
import numpy as np
import pytest

from tests import kv_reference as ref

pytestmark = pytest.mark.gpu
E_RANGE = -5


@pytest.fixture(scope="module")
def fl():
    import torch
    from fuselink_amd import core, kv
    core.init(0)
    return core, kv, torch


def dev(torch, a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a))
    return (t if dtype is None else t.to(dtype)).cuda()


def held(cache, T, H, D):
    return ref.unpack(cache.pages.cpu().numpy(), T, H, D)


def same_numbers(got, exp, what):
    np.testing.assert_array_equal(np.isnan(got), np.isnan(exp), err_msg=what)
    np.testing.assert_array_equal(np.nan_to_num(got), np.nan_to_num(exp), err_msg=what)   # -0 equals 0


def same_cache(got, exp, what=""):
    for name in ("s", "k", "v", "low", "high"):
        same_numbers(got[name], exp[name], f"{what} {name}")


def tables(rng, lens, T, spare=0, width=None):
    """Page tables over a pool in a random order, with unused pages between; unused entries are -1."""
    need = [-(-x // T) + spare for x in lens]
    n = sum(need) + 2
    order = rng.permutation(n)
    width = max(max(need), 1) if width is None else width
    t, at = np.full((len(lens), width), -1, np.int32), 0
    for b, m in enumerate(need):
        t[b, :m] = order[at:at + m]
        at += m
    return t, n


def make(fl, rng, lens, T, H, D, spread=1.0, fill=0xAA):
    """A cache filled by the reference itself, as records on the device: (cache, dict, table).  Unused bytes are `fill`."""
    core, kv, torch = fl
    table, n = tables(rng, lens, T)
    c = ref.empty(n, T, H, D)
    starts = np.concatenate([[0], np.cumsum(lens)]).astype(int)
    gain = np.exp(spread * rng.standard_normal((1, H, D)))
    k = (rng.standard_normal((starts[-1], H, D)) * gain).astype(np.float32).astype(np.float64)
    v = (rng.standard_normal((starts[-1], H, D)) * np.exp(spread * rng.standard_normal((starts[-1], H, 1)))).astype(np.float32).astype(np.float64)
    ref.store(c, k, v, table, [0] * len(lens), starts)
    return records(fl, c, T, H, D, lens, table, fill), c, table


def records(fl, c, T, H, D, lens, table, fill=0xAA):
    core, kv, torch = fl
    n = c["k"].shape[0]
    back = {float(x): i for i, x in reversed(list(enumerate(ref.CODES))) if not np.isnan(x)}
    to_code = np.vectorize(lambda x: 0x7f if np.isnan(x) else back[float(x)], otypes=[np.uint8])
    raw = np.full((n, ref.page_bytes(T, H, D)), fill, np.uint8)
    a = H * T * D
    kc, vc = to_code(c["k"]), to_code(c["v"])
    # slots that hold nothing are anything at all: here the code of NaN
    live = np.zeros((n, T), bool)
    for b, x in enumerate(lens):
        for p in range(x):
            live[table[b][p // T], p % T] = True
    for codes in (kc, vc):
        codes.transpose(0, 2, 1, 3)[~live] = 0x7f
    raw[:, :a], raw[:, a:2 * a] = kc.reshape(n, -1), vc.reshape(n, -1)
    raw[:, 2 * a:2 * a + H * D] = c["low"].reshape(n, -1).view(np.uint8)
    raw[:, 2 * a + H * D:2 * a + 2 * H * D] = c["high"].reshape(n, -1).view(np.uint8)
    raw[:, 2 * a + 2 * H * D:2 * a + 2 * H * D + 8 * H] = np.ascontiguousarray(c["s"].astype(np.float32)).reshape(n, -1).view(np.uint8)
    return kv.PageCache(dev(torch, raw), tokens=T, heads=H, dim=D)


# ---- store ----------------------------------------------------------------------------------------------------------
STORE = [  # T, H, D, tokens held before, new ones
    (16, 2, 128, [0], [1]), (16, 8, 128, [0, 0, 0], [16, 17, 40]), (16, 1, 64, [15, 16, 17], [1, 1, 1]), (32, 3, 80, [5, 0, 31], [0, 70, 2]),
    (48, 2, 96, [47, 20], [2, 100]), (64, 1, 256, [10, 0], [60, 129]), (256, 2, 128, [0, 250], [256, 20]), (256, 1, 256, [100], [300]),
    (16, 5, 16, [3, 0], [30, 7]), (128, 1, 48, [0, 1, 127], [128, 127, 2]),
]


@pytest.mark.parametrize("case", STORE, ids=str)
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp32"])
def test_store(fl, case, kind):
    core, kv, torch = fl
    T, H, D, had, new = case
    dt = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[kind]
    rng = np.random.default_rng(T + D + sum(new))
    B = len(had)
    total = [a + b for a, b in zip(had, new)]
    cache, c, table = make(fl, rng, had, T, H, D, fill=0)
    need = max(-(-max(total) // T), 1)
    pool = torch.zeros(c["k"].shape[0] + B * need, ref.page_bytes(T, H, D), dtype=torch.uint8, device="cuda")
    pool[:cache.pages.shape[0]] = cache.pages
    full, at = np.full((B, need), -1, np.int32), cache.pages.shape[0]
    for b in range(B):
        m = -(-had[b] // T)
        full[b, :m] = table[b, :m]
        for j in range(m, -(-total[b] // T)):
            full[b, j] = at
            at += 1
    cache = kv.PageCache(pool, T, H, D)
    before = held(cache, T, H, D)
    pad = 2                                               # tokens of the call that are nobody's
    starts = pad + np.concatenate([[0], np.cumsum(new)])
    n = int(starts[-1]) + pad
    k, v = (dev(torch, rng.standard_normal((n, H, D)) * np.exp(2 * rng.standard_normal((n, H, 1))), torch.float32).to(dt) for _ in range(2))
    status = core.new_status()
    kv.store(cache, k, v, dev(torch, full), dev(torch, np.array(had, np.int32)), status, starts=dev(torch, starts.astype(np.int32)))
    torch.cuda.synchronize()
    assert int(status) == 0
    exp = {x: y.copy() for x, y in before.items()}
    ref.store(exp, k.cpu().double().numpy(), v.cpu().double().numpy(), full, had, starts)
    same_cache(held(cache, T, H, D), exp)


@pytest.mark.parametrize("tokens,dim", [(16, 32), (64, 32), (16, 256), (64, 128), (128, 144), (128, 256)])
def test_store_values_at_the_edges(fl, tokens, dim):
    """Blocks of zeros, numbers that are not finite, the largest and smallest of a type, magnitudes at 448 * 2^e."""
    core, kv, torch = fl
    T, H, D = tokens, 2, dim
    n = 16 * 8
    x = np.zeros((n, H, D))
    rng = np.random.default_rng(0)
    x[0:16] = 0
    x[16:32] = rng.standard_normal((16, H, D)); x[16, 0, 0], x[17, 0, 1], x[18, 1, 2] = np.nan, np.inf, -np.inf
    x[32:48] = rng.standard_normal((16, H, D)) * 1e38
    x[48:64] = rng.standard_normal((16, H, D)) * 1e-40
    x[64:80] = rng.uniform(-1, 1, (16, H, D)); x[64, 0, 0], x[65, 1, 1] = 448.0, -448.0 * 2 ** -9
    x[80:96] = rng.uniform(-1, 1, (16, H, D)); x[80, 0, 0], x[81, 1, 1] = np.nextafter(np.float32(448), np.float32(500)), np.nextafter(np.float32(1.75), np.float32(2))
    x[96:112] = np.nan
    x[112:128] = rng.standard_normal((16, H, D)) * np.exp(8 * rng.standard_normal((16, H, D)))
    with np.errstate(over="ignore"):        # what passes the largest number becomes an infinity, one more value to test
        x = x.astype(np.float32)
    cache = kv.PageCache(torch.full((9, kv.page_bytes(T, H, D)), 0xA5, dtype=torch.uint8, device="cuda"), T, H, D)
    table = np.array([[7, 3, 1, 0, 8, 2, 5, 4]], np.int32)
    exp = held(cache, T, H, D)
    status = core.new_status()
    kv.store(cache, dev(torch, x), dev(torch, -x), dev(torch, table), dev(torch, np.zeros(1, np.int32)), status)
    ref.store(exp, x.astype(np.float64), -x.astype(np.float64), table, [0], [0, n])
    torch.cuda.synchronize()
    assert int(status) == 0
    same_cache(held(cache, T, H, D), exp)


@pytest.mark.parametrize("shift", [0, 1])
def test_store_strided(fl, shift):
    """Keys and values as slices of one projection's output, aligned to 16 bytes and not."""
    core, kv, torch = fl
    T, H, D, n = 16, 3, 64, 37
    rng = np.random.default_rng(shift)
    qkv = dev(torch, rng.standard_normal((n, 3 * H * D + 8)), torch.float32).to(torch.bfloat16)
    k = qkv[:, H * D + shift:2 * H * D + shift].unflatten(1, (H, D))
    v = qkv[:, 2 * H * D + shift:3 * H * D + shift].unflatten(1, (H, D))
    wide = torch.zeros(4, 2, kv.page_bytes(T, H, D), dtype=torch.uint8, device="cuda")   # two layers share a page
    cache = kv.PageCache(wide[:, 1], T, H, D)
    exp = ref.empty(4, T, H, D)
    table = np.array([[2, 0, 3]], np.int32)
    status = core.new_status()
    kv.store(cache, k, v, dev(torch, table), dev(torch, np.zeros(1, np.int32)), status)
    ref.store(exp, k.cpu().double().numpy(), v.cpu().double().numpy(), table, [0], [0, n])
    torch.cuda.synchronize()
    assert int(status) == 0 and int(wide[:, 0].sum()) == 0
    same_cache(held(cache, T, H, D), exp)


def test_store_token_by_token(fl):
    """One token at a time, as decoding does: scales only grow, codes follow them, bounds are those of what is held."""
    core, kv, torch = fl
    T, H, D, B, n = 16, 2, 80, 3, 35
    rng = np.random.default_rng(5)
    x = rng.standard_normal((n, B, H, D)) * np.exp(1.5 * rng.standard_normal((n, B, H, 1)))
    x = dev(torch, x, torch.float32).to(torch.float16)
    table, pages = tables(rng, [n] * B, T)
    cache = kv.PageCache(torch.zeros(pages, kv.page_bytes(T, H, D), dtype=torch.uint8, device="cuda"), T, H, D)
    exp, status, lens = ref.empty(pages, T, H, D), core.new_status(), torch.zeros(B, dtype=torch.int32, device="cuda")
    for i in range(n):
        kv.store(cache, x[i], x[i] * 2, dev(torch, table), lens, status)
        lens += 1
        y = x[i].cpu().double().numpy()
        ref.store(exp, y, (x[i] * 2).cpu().double().numpy(), table, [i] * B, list(range(B + 1)))
    torch.cuda.synchronize()
    assert int(status) == 0
    same_cache(held(cache, T, H, D), exp)


# ---- attention ------------------------------------------------------------------------------------------------------
def run_attend(fl, T, H, G, D, lens, news, kind, causal=True, weights=False, spread=0.7, scale=None, nobody=1, seed=0, table_width=None):
    core, kv, torch = fl
    dt = {"bf16": torch.bfloat16, "fp16": torch.float16}[kind]
    rng = np.random.default_rng(seed + T * 7 + D + sum(lens))
    cache, c, table = make(fl, rng, lens, T, H, D, spread)
    starts = nobody + np.concatenate([[0], np.cumsum(news)])
    n = int(starts[-1]) + nobody
    q = dev(torch, rng.standard_normal((n, H * G, D)), torch.float32).to(dt)
    out = torch.full_like(q, 7.0)
    lse = torch.full((n, H * G), 7.0, device="cuda")
    w0 = w1 = None
    if weights:
        w0 = dev(torch, rng.uniform(0, 2, (len(lens), H, max(lens) + 5)).astype(np.float32))
        w1 = torch.full_like(w0, -1.0)
    status = core.new_status()
    got = kv.attend(cache, q, dev(torch, table), dev(torch, np.array(lens, np.int32)), status, starts=dev(torch, starts.astype(np.int32)), causal=causal,
                    scale=scale, out=out, lse=lse, weights=w1, weights_in=w0)
    torch.cuda.synchronize()
    assert got is out and int(status) == 0
    r = ref.attend(c, q.cpu().double().numpy(), table, lens, starts, 1 / np.sqrt(D) if scale is None else scale, causal)
    check_out(torch, out, lse, r, dt, lens, starts)
    if weights:
        w = w1.cpu().double().numpy()
        for b, x in enumerate(lens):
            base = w0[b].cpu().double().numpy()
            tol = r["wslack"][b] * 1.1 + (r["weights"][b] + base[:, :x]) * (max(news) * G + 64) * 2.0 ** -23
            assert (np.abs(w[b, :, :x] - base[:, :x] - r["weights"][b]) <= tol).all()
            np.testing.assert_array_equal(w[b, :, x:], base[:, x:])


def check_out(torch, out, lse, r, dt, lens, starts):
    n = out.shape[0]
    mine = np.zeros(n, bool)
    mine[starts[0]:starts[-1]] = True
    o = out.cpu().double().numpy()
    assert (o[~mine] == 7).all(), "tokens of no sequence were written"
    tol = ref.out_tolerance(r, torch.finfo(dt).eps, max(lens))
    bad = ~(np.abs(o - r["out"]) <= tol) & mine[:, None, None]
    assert not bad.any(), f"{int(bad.sum())} outputs off, worst {np.abs(o - r['out'])[bad].max()} at {np.argwhere(bad)[0]}"
    if lse is not None:
        l = lse.cpu().double().numpy()
        assert (l[~mine] == 7).all()
        fin = np.isfinite(r["lse"]) & mine[:, None]
        assert (l[mine[:, None] & ~np.isfinite(r["lse"])] == -np.inf).all()
        e = np.where(fin, r["lse"], 0.0)
        assert (np.abs(np.where(fin, l, 0.0) - e) <= r["slack"] * 1.1 + (np.abs(e) + 16 + max(lens) * 0.5) * 2.0 ** -22).all()


ATTEND = [  # T, H, G, D, lens, query tokens
    (16, 2, 4, 128, [1], [1]), (16, 2, 4, 128, [16, 17, 33], [1, 1, 1]), (16, 1, 8, 64, [31, 200, 5], [1, 1, 1]), (32, 3, 1, 128, [100, 0, 64], [1, 1, 1]),
    (48, 2, 7, 80, [97, 48], [1, 1]), (64, 1, 16, 256, [130, 63], [1, 1]), (256, 1, 5, 96, [300, 256], [1, 1]), (16, 2, 20, 128, [70, 9], [1, 1]),
    (16, 2, 40, 64, [70], [1]), (16, 1, 2, 16, [40], [3]), (16, 1, 2, 48, [600, 33], [1, 1]), (16, 2, 4, 128, [50, 20, 7], [5, 20, 7]),
    (32, 1, 4, 128, [90, 33], [33, 16]), (16, 1, 3, 64, [150, 40], [70, 40]), (16, 1, 1, 112, [200], [130]), (64, 1, 2, 256, [100, 64], [50, 64]),
    (128, 2, 1, 144, [129], [100]), (16, 1, 4, 128, [3, 10], [9, 10]), (16, 1, 1, 128, [2100], [1]),
    (16, 1, 2, 64, [9000], [1]), (16, 1, 2, 128, list(range(0, 70)), [1] * 70), (16, 1, 4, 64, [(37 * i) % 90 for i in range(70)], [(5 * i) % 11 for i in range(70)]),
    (32, 1, 2, 80, [700, 40], [90, 40]), (16, 1, 8, 128, [1100], [40]), (16, 2, 4, 128, [1500, 700], [20, 9]), (16, 1, 2, 256, [1200], [20]),
    (16, 1, 4, 64, [2000, 30], [31, 30]), (48, 1, 6, 256, [1000], [50]),
]


@pytest.mark.parametrize("case", ATTEND, ids=str)
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("causal", [True, False])
def test_attend(fl, case, kind, causal):
    T, H, G, D, lens, news = case
    run_attend(fl, T, H, G, D, lens, news, kind, causal)


@pytest.mark.parametrize("case", ATTEND, ids=str)
def test_attend_weights(fl, case):
    T, H, G, D, lens, news = case
    run_attend(fl, T, H, G, D, lens, news, "bf16", weights=True)


MANY = [  # more than 128 tiles of 128 rows
    (16, 65, 1, 112, [200], [130]), (16, 65, 3, 64, [150, 40], [70, 40]), (32, 43, 2, 80, [700, 40], [90, 40]), (16, 65, 4, 128, [600], [40]),
    (16, 1, 4, 64, [33 + (7 * i) % 60 for i in range(70)], [33] * 70), (48, 66, 1, 128, [150, 0, 260], [150, 0, 250]),
]


@pytest.mark.parametrize("case", MANY, ids=str)
@pytest.mark.parametrize("kind,causal,weights", [("bf16", True, True), ("fp16", False, False)])
def test_attend_many_tiles(fl, case, kind, causal, weights):
    T, H, G, D, lens, news = case
    run_attend(fl, T, H, G, D, lens, news, kind, causal, weights=weights)


@pytest.mark.parametrize("n,H", [(3, 2), (5, 2), (20, 2), (40, 2), (40, 65)])
def test_attend_nan_is_seen_by_those_who_may(fl, n, H):
    """A NaN among the values reaches exactly the queries that see its token; one among the keys likewise, whole rows."""
    core, kv, torch = fl
    T, G, D, x = 16, 4, 64, 40
    rng = np.random.default_rng(3)
    for side in (1, 0):
        cache, c, table = make(fl, rng, [x], T, H, D)
        late = min(9, n - 1)               # the last `late` queries see the token
        at = x - late
        raw = cache.pages
        off = side * H * T * D + (1 * T + at % T) * D + 5
        raw[int(table[0, at // T]), off] = 0x7f
        c["kv"[side]][table[0, at // T], 1, at % T, 5] = np.nan
        q = dev(torch, rng.standard_normal((n, H * G, D)), torch.float32).to(torch.bfloat16)
        status = core.new_status()
        out = kv.attend(cache, q, dev(torch, table), dev(torch, np.array([x], np.int32)), status)
        torch.cuda.synchronize()
        with np.errstate(invalid="ignore"):
            r = ref.attend(c, q.cpu().double().numpy(), table, [x], [0, n], 1 / np.sqrt(D))
        o = out.cpu().double().numpy()
        nan = np.zeros(o.shape, bool)
        if side:
            nan[n - late:, G:2 * G, 5] = True
        else:
            nan[n - late:, G:2 * G, :] = True
        np.testing.assert_array_equal(np.isnan(o), nan)
        tol = ref.out_tolerance(r, torch.finfo(torch.bfloat16).eps, x)
        assert (np.abs(o - r["out"])[~nan] <= tol[~nan]).all()


@pytest.mark.parametrize("T", [16, 32])
def test_attend_scales_far_apart(fl, T):
    """Blocks whose value scales differ by powers of two up to 2^12 within a step of 32 keys and 2^60 beyond it."""
    core, kv, torch = fl
    H, G, D, x = 1, 4, 64, 16 * T
    rng = np.random.default_rng(T)
    k, v = rng.standard_normal((x, H, D)), rng.standard_normal((x, H, D))
    for j in range(16):
        v[j * T:(j + 1) * T] *= 2.0 ** ((0, -12, 30, 18, -30, -20, 5, 0)[j % 8])
    table, pages = tables(rng, [x], T)
    c = ref.empty(pages, T, H, D)
    ref.store(c, k, v, table, [0], [0, x])
    cache = records(fl, c, T, H, D, [x], table)
    q = dev(torch, rng.standard_normal((1, G, D)) * 4, torch.float32).to(torch.float16)
    out = kv.attend(cache, q.expand(1, G, D), dev(torch, table), dev(torch, np.array([x], np.int32)), core.new_status()).cpu().double().numpy()
    r = ref.attend(c, q.cpu().double().numpy(), table, [x], [0, 1], 1 / np.sqrt(D))
    # what is computed lies within tol of the definition before it becomes 16 bits wide; from 65520 on that is infinity
    tol = ref.out_tolerance(r, torch.finfo(torch.float16).eps, x)
    low, high = np.abs(r["out"]) - tol, np.abs(r["out"]) + tol
    assert (np.abs(out - r["out"])[high < 65504] <= tol[high < 65504]).all() and np.isinf(out[low > 65520]).all() and not np.isnan(out).any()


@pytest.mark.parametrize("scale", [0.0, -0.3, 40.0])
def test_attend_scale(fl, scale):
    run_attend(fl, 16, 2, 4, 64, [77, 20], [1, 20], "bf16", scale=scale, weights=True)


@pytest.mark.parametrize("H,lens,n", [(2, [50, 21, 33], 2), (22, [150, 121, 133], 70)], ids=str)
def test_attend_strided_and_uniform(fl, H, lens, n):
    """Queries and outputs inside wider tensors, at odd offsets; no starts: every sequence has equally many tokens."""
    core, kv, torch = fl
    T, G, D = 16, 2, 64
    starts = [0, n, 2 * n, 3 * n]
    rng = np.random.default_rng(9)
    cache, c, table = make(fl, rng, lens, T, H, D)
    for shift in (0, 1, 4):
        wide = dev(torch, rng.standard_normal((len(lens) * n, H * G + 1, D + 8)), torch.float32).to(torch.float16)
        q = wide[:, 1:, shift:shift + D]
        res = torch.full((H * G, len(lens) * n, D + 8), 7.0, dtype=torch.float16, device="cuda")
        out = res.transpose(0, 1)[:, :, shift:shift + D]
        wide_table = torch.full((len(lens), table.shape[1] + 3), -1, dtype=torch.int32, device="cuda")
        wide_table[:, :table.shape[1]] = dev(torch, table)
        status = core.new_status()
        kv.attend(cache, q, wide_table[:, :table.shape[1]], dev(torch, np.array(lens, np.int32)), status, out=out)
        torch.cuda.synchronize()
        assert int(status) == 0
        r = ref.attend(c, q.cpu().double().numpy(), table, lens, starts, 1 / np.sqrt(D))
        check_out(torch, out, None, r, torch.float16, lens, starts)
        assert (res[:, :, :shift] == 7).all() and (res[:, :, shift + D:] == 7).all()


@pytest.mark.parametrize("n,x,H", [(1, 50, 2), (1, 5000, 2), (3, 50, 2), (20, 1500, 2), (40, 90, 2), (40, 90, 65), (40, 400, 65)])
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_attend_queries_that_are_not_finite(fl, n, x, H, kind):
    """A NaN or an infinity in a query makes its own row NaN -- with keys of both signs an infinite channel gives an
    infinite largest score -- and touches no other row."""
    core, kv, torch = fl
    T, G, D = 16, 4, 128
    rng = np.random.default_rng(n + x)
    cache, c, table = make(fl, rng, [x], T, H, D)
    q = dev(torch, rng.standard_normal((n, H * G, D)), torch.float32).to({"bf16": torch.bfloat16, "fp16": torch.float16}[kind])
    bad = np.zeros((n, H * G), bool)
    for i, (t, h, value) in enumerate([(0, 1, np.nan), (n // 2, 2, np.inf), (n - 1, 6, -np.inf)]):
        q[t, h, 17 * i + 3] = value
        bad[t, h] = True
    status, lse = core.new_status(), torch.zeros(n, H * G, device="cuda")
    out = kv.attend(cache, q, dev(torch, table), dev(torch, np.array([x], np.int32)), status, lse=lse)
    r = ref.attend(c, np.where(bad[:, :, None], 0, q.cpu().double().numpy()), table, [x], [0, n], 1 / np.sqrt(D))
    o, s = out.cpu().double().numpy(), lse.cpu().double().numpy()
    assert int(status) == 0 and np.isnan(o[bad]).all() and np.isnan(s[bad]).all()
    assert (np.abs(o - r["out"]) <= ref.out_tolerance(r, torch.finfo(out.dtype).eps, x))[~bad].all()


@pytest.mark.parametrize("n,x,H", [(1, 50, 1), (1, 5000, 1), (3, 50, 1), (20, 90, 1), (40, 1500, 1), (40, 300, 65)])
def test_attend_scores_that_are_all_minus_infinity(fl, n, x, H):
    """Such a row draws nothing from any key: zeros, a log-sum of -inf, and the others' weights as without it."""
    core, kv, torch = fl
    T, G, D = 16, 4, 64
    rng = np.random.default_rng(n + x)
    cache = kv.PageCache(torch.zeros(-(-x // T), kv.page_bytes(T, H, D), dtype=torch.uint8, device="cuda"), T, H, D)
    k, v = (dev(torch, rng.uniform(0.5, 1, (x, H, D)), torch.float32) for _ in range(2))
    table, lens, status = dev(torch, np.arange(-(-x // T), dtype=np.int32)[None]), dev(torch, np.array([x], np.int32)), core.new_status()
    kv.store(cache, k, v, table, torch.zeros_like(lens), status)
    q = dev(torch, rng.standard_normal((n, H * G, D)), torch.float32).to(torch.bfloat16)
    c = ref.unpack(cache.pages.cpu().numpy(), T, H, D)
    r = ref.attend(c, q.cpu().double().numpy(), table.cpu().numpy(), [x], [0, n], 1 / np.sqrt(D))
    q[n - 1, 1, 3] = -np.inf
    lse, w = torch.zeros(n, H * G, device="cuda"), torch.zeros(1, H, x, device="cuda")
    out = kv.attend(cache, q, table, lens, status, lse=lse, weights=w)
    assert int(status) == 0 and int(out[n - 1, 1].abs().sum()) == 0 and float(lse[n - 1, 1]) == -np.inf
    others = np.arange(n * H * G) != (n - 1) * H * G + 1
    e = np.abs(out.cpu().double().numpy() - r["out"]) <= ref.out_tolerance(r, torch.finfo(out.dtype).eps, x)
    assert e.reshape(n * H * G, D)[others].all()
    assert not w.isnan().any() and abs(float(w.double().sum()) - (n * H * G - 1)) <= 1e-3 * n * H * G   # (each row's sum is 1 within the 2^-11 of its log-sum)


def test_views_that_overlap(fl):
    """What a call writes may lie between what it reads, but not on it."""
    core, kv, torch = fl
    T, H, G, D, x = 16, 2, 4, 64, 40
    rng = np.random.default_rng(2)
    cache, c, table = make(fl, rng, [x, x], T, H, D)
    wide = dev(torch, rng.standard_normal((2, 2 * H * G * D)), torch.float32).to(torch.bfloat16)
    q, between = (wide[:, i * H * G * D:(i + 1) * H * G * D].unflatten(1, (H * G, D)) for i in (0, 1))
    args = dev(torch, table), dev(torch, np.array([x, x], np.int32)), core.new_status()
    exp = kv.attend(cache, q, *args)
    for out in (q, wide[:, D:D + H * G * D].unflatten(1, (H * G, D)), wide.view(-1)[8:8 + 2 * H * G * D].view(2, H * G, D)):
        with pytest.raises(ValueError, match="overlaps q"):
            kv.attend(cache, q, *args, out=out)
    kv.attend(cache, q, *args, out=between)
    assert torch.equal(between, exp)
    w = torch.zeros(2, H, 2 * 64, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        kv.attend(cache, q, *args, weights=w[:, :, :64], weights_in=w[:, :, 1:65])
    kv.attend(cache, q, *args, weights=w[:, :, :64], weights_in=w[:, :, :64])
    to = kv.PageCache(torch.zeros(4, kv.page_bytes(T, H, D), dtype=torch.uint8, device="cuda"), T, H, D)
    to_table = dev(torch, np.arange(4, dtype=np.int32).reshape(2, 2))
    with pytest.raises(ValueError, match="overlaps weights"):
        kv.evict(cache, args[0], args[1], w[:, :, :64], 20, to, to_table, args[2], new_weights=w[:, :, 40:104])
    assert int(args[2]) == 0


def test_pool_past_four_gigabytes(fl):
    """Pages at the far end of a pool of 4.5 GiB: store, attention, the choice of pages and eviction."""
    core, kv, torch = fl
    T, H, G, D, x = 16, 8, 2, 128, 150
    pb = kv.page_bytes(T, H, D)
    n = (9 << 29) // pb
    cache = kv.PageCache(torch.empty(n, pb, dtype=torch.uint8, device="cuda"), T, H, D)
    rng = np.random.default_rng(8)
    table = np.array([list(range(n - 1, n - 6, -1)) + list(range(5))], np.int32)
    k, v = (dev(torch, rng.standard_normal((x, H, D)), torch.float32) for _ in range(2))
    status, lens = core.new_status(), dev(torch, np.array([x], np.int32))
    kv.store(cache, k, v, dev(torch, table), torch.zeros_like(lens), status)
    c = ref.empty(10, T, H, D)
    small = np.arange(10, dtype=np.int32)[None]
    ref.store(c, k.cpu().double().numpy(), v.cpu().double().numpy(), small, [0], [0, x])
    got = ref.unpack(cache.pages[dev(torch, table[0]).long()].cpu().numpy(), T, H, D)
    same_cache(got, c)
    q = dev(torch, rng.standard_normal((1, H * G, D)), torch.float32).to(torch.bfloat16)
    out = kv.attend(cache, q, dev(torch, table), lens, status)
    check_out(torch, out, None, ref.attend(c, q.cpu().double().numpy(), small, [x], [0, 1], 1 / np.sqrt(D)), torch.bfloat16, [x], [0, 1])
    sel = kv.select_pages(cache, q, dev(torch, table), lens, 4, status)
    np.testing.assert_array_equal(sel.cpu().numpy(), ref.select(c, q.cpu().double().numpy(), small, [x], [0, 1], 4, 1, 1))
    w = dev(torch, rng.random((1, H, x)).astype(np.float32))
    to_table = np.array([[n // 2, n - 7, n - 9]], np.int32)
    kept, _, _ = kv.evict(cache, dev(torch, table), lens, w, 40, cache, dev(torch, to_table), status)
    exp = ref.empty(3, T, H, D)
    k_exp, _ = ref.evict(c, small, [x], w.cpu().numpy(), 40, 0, 0, exp, np.arange(3)[None])
    np.testing.assert_array_equal(kept.cpu().numpy(), k_exp)
    same_cache(ref.unpack(cache.pages[dev(torch, to_table[0]).long()].cpu().numpy(), T, H, D), exp)
    assert int(status) == 0


# ---- selected pages -------------------------------------------------------------------------------------------------
SELECT = [  # T, H, G, D, lens, query tokens, count, first, last
    (16, 2, 4, 128, [500], [1], 4, 1, 1), (16, 2, 4, 128, [16, 17, 900], [1, 1, 1], 8, 0, 1), (32, 3, 1, 64, [700, 33], [3, 5], 5, 2, 2),
    (48, 1, 7, 80, [2000, 0], [1, 0], 9, 0, 0), (48, 2, 4, 128, [3, 200, 1900], [1, 1, 1], 45, 1, 1), (16, 1, 2, 96, [40, 3000], [30, 6], 200, 0, 1), (16, 1, 20, 96, [1500], [2], 6, 1, 2), (64, 1, 16, 256, [3000], [1], 10, 1, 1),
    (16, 2, 2, 16, [300, 40], [40, 40], 3, 0, 1), (16, 1, 1, 128, [20000], [1], 64, 1, 1), (256, 1, 2, 48, [5000], [1], 7, 0, 3),
]


@pytest.mark.parametrize("case", SELECT, ids=str)
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_select_and_attend(fl, case, kind):
    core, kv, torch = fl
    T, H, G, D, lens, news, count, first, last = case
    dt = {"bf16": torch.bfloat16, "fp16": torch.float16}[kind]
    rng = np.random.default_rng(sum(lens) + count)
    cache, c, table = make(fl, rng, lens, T, H, D, 0.7)
    starts = 1 + np.concatenate([[0], np.cumsum(news)])
    n = int(starts[-1]) + 1
    q = dev(torch, rng.standard_normal((n, H * G, D)), torch.float32).to(dt)
    status = core.new_status()
    d_table, d_lens, d_starts = dev(torch, table), dev(torch, np.array(lens, np.int32)), dev(torch, starts.astype(np.int32))
    for causal in (True, False):
        sel = torch.full((n, H, count), -7, dtype=torch.int32, device="cuda")
        kv.select_pages(cache, q, d_table, d_lens, count, status, starts=d_starts, first=first, last=last, causal=causal, out=sel)
        exp = ref.select(c, q.cpu().double().numpy(), table, lens, starts, count, first, last, causal)
        exp[0], exp[-1] = -7, -7
        np.testing.assert_array_equal(sel.cpu().numpy(), exp)
        out = torch.full_like(q, 7.0)
        lse = torch.full((n, H * G), 7.0, device="cuda")
        kv.attend(cache, q, d_table, d_lens, status, starts=d_starts, selected=sel, causal=causal, out=out, lse=lse)
        torch.cuda.synchronize()
        assert int(status) == 0
        r = ref.attend(c, q.cpu().double().numpy(), table, lens, starts, 1 / np.sqrt(D), causal, selected=exp)
        check_out(torch, out, lse, r, dt, lens, starts)


def test_select_ties_and_odd_queries(fl):
    """Equal pages take the lower index; queries of zeros, of NaN and infinities count what is left of them."""
    core, kv, torch = fl
    T, H, G, D, x = 16, 1, 2, 64, 16 * 300
    rng = np.random.default_rng(1)
    cache, c, table = make(fl, rng, [x], T, H, D)
    table = table[:, rng.integers(0, 5, 300)].astype(np.int32)       # five pages, again and again
    for kind in range(4):
        qn = rng.standard_normal((1, H * G, D)).astype(np.float32)
        if kind == 1:
            qn[:] = 0
        if kind == 2:
            qn[0, 0, 3], qn[0, 1, 7], qn[0, 1, 8] = np.nan, np.inf, -np.inf
        if kind == 3:
            qn[:] = np.nan
        q = dev(torch, qn).to(torch.float16)
        status = core.new_status()
        got = kv.select_pages(cache, q, dev(torch, table), dev(torch, np.array([x], np.int32)), 70, status, first=2, last=1)
        np.testing.assert_array_equal(got.cpu().numpy(), ref.select(c, q.cpu().double().numpy(), table, [x], [0, 1], 70, 2, 1))
        assert int(status) == 0


def test_select_among_very_many(fl):
    """More pages than a workgroup keeps keys of, few of them different."""
    core, kv, torch = fl
    T, H, G, D, n = 16, 1, 1, 32, 17001
    rng = np.random.default_rng(1)
    cache, c, table = make(fl, rng, [16 * 40], T, H, D)
    table = table[:, rng.integers(0, 40, n)].astype(np.int32)
    q = dev(torch, rng.standard_normal((1, H * G, D)), torch.float32).to(torch.bfloat16)
    status = core.new_status()
    for count in (100, 1000, 16999):
        got = kv.select_pages(cache, q, dev(torch, table), dev(torch, np.array([16 * n - 3], np.int32)), count, status, first=3, last=7)
        np.testing.assert_array_equal(got.cpu().numpy(), ref.select(c, q.cpu().double().numpy(), table, [16 * n - 3], [0, 1], count, 3, 7))
    assert int(status) == 0


# ---- eviction -------------------------------------------------------------------------------------------------------
EVICT = [  # T, T of the new pages, H, D, lens, budget, first, recent
    (16, 16, 2, 64, [100, 40, 41], 40, 4, 8), (16, 32, 1, 80, [300, 0, 1], 33, 0, 0), (32, 16, 3, 128, [200], 100, 0, 100), (256, 48, 1, 256, [700], 300, 2, 5),
    (16, 16, 1, 16, [2500, 1100], 1029, 1, 28), (16, 256, 2, 128, [600, 16], 1, 0, 1), (48, 16, 1, 96, [50], 64, 64, 0), (16, 128, 1, 256, [9000], 260, 3, 3),
    (16, 64, 3, 128, [500, 70], 150, 4, 8), (32, 256, 1, 256, [700, 40], 520, 1, 9),
    (64, 64, 1, 16, [17000, 16384, 16385], 5000, 2, 9), (16, 16, 1, 16, [(i * 13) % 80 for i in range(70)], 30, 1, 2),
]


@pytest.mark.parametrize("case", EVICT, ids=str)
@pytest.mark.parametrize("kind", ["spread", "ties", "odd"])
def test_evict(fl, case, kind):
    core, kv, torch = fl
    T, T2, H, D, lens, budget, first, recent = case
    rng = np.random.default_rng(sum(lens) + budget)
    cache, c, table = make(fl, rng, lens, T, H, D)
    w = np.exp(2 * rng.standard_normal((len(lens), H, max(lens) + 3))).astype(np.float32)
    if kind == "ties":
        w = rng.integers(0, 3, w.shape).astype(np.float32) * np.where(rng.random(w.shape) < 0.5, -0.0, 1.0).astype(np.float32)
    if kind == "odd":
        w = (rng.standard_normal(w.shape) * 10.0 ** rng.integers(-44, 38, w.shape)).astype(np.float32)
        w[rng.random(w.shape) < 0.2] = np.nan
        w[rng.random(w.shape) < 0.1] = np.inf
        w[rng.random(w.shape) < 0.1] = -np.inf
    per = -(-budget // T2)
    n2 = per * len(lens) + 1
    table2 = rng.permutation(n2)[:per * len(lens)].reshape(len(lens), per).astype(np.int32)
    to = kv.PageCache(torch.full((n2, kv.page_bytes(T2, H, D)), 0xA5, dtype=torch.uint8, device="cuda"), T2, H, D)
    exp = held(to, T2, H, D)
    status = core.new_status()
    nw = torch.full((len(lens), H, budget + 2), -3.0, device="cuda")
    kept, nw, nl = kv.evict(cache, dev(torch, table), dev(torch, np.array(lens, np.int32)), dev(torch, w), budget, to, dev(torch, table2), status,
                            first=first, recent=recent, new_weights=nw)
    torch.cuda.synchronize()
    assert int(status) == 0
    k, x = ref.evict(c, table, lens, w, budget, first, recent, exp, table2)
    np.testing.assert_array_equal(kept.cpu().numpy(), k)
    np.testing.assert_array_equal(nl.cpu().numpy(), np.minimum(lens, budget))
    same_numbers(nw.cpu().double().numpy()[:, :, :budget], x, "weights")
    assert (nw[:, :, budget:] == 0).all()
    same_cache(held(to, T2, H, D), exp)


# ---- what is wrong with device-resident numbers ---------------------------------------------------------------------
def test_bad_pages(fl):
    """A page number outside the pool: reported, not written, its keys not seen; all else as if it were absent."""
    core, kv, torch = fl
    T, H, G, D, lens = 16, 2, 2, 64, [100, 60]
    for wrong in (-1, -2 ** 31, 10 ** 6, 2 ** 31 - 1):
        rng = np.random.default_rng(2)
        cache, c, table = make(fl, rng, lens, T, H, D)
        bad = table.copy()
        bad[0, 2] = wrong
        d_bad, d_lens = dev(torch, bad), dev(torch, np.array(lens, np.int32))
        q = dev(torch, rng.standard_normal((2, H * G, D)), torch.float32).to(torch.bfloat16)
        status = core.new_status()
        out = kv.attend(cache, q, d_bad, d_lens, status)
        torch.cuda.synchronize()
        assert int(status) == E_RANGE
        seen = [[j for j in range(7) if j != 2], list(range(4))]
        pick = np.full((2, H, 7), -1)
        for b in range(2):
            pick[b, :, :len(seen[b])] = seen[b]
        r = ref.attend(c, q.cpu().double().numpy(), table, lens, [0, 1, 2], 1 / np.sqrt(D), selected=pick)
        check_out(torch, out, None, r, torch.bfloat16, lens, [0, 1, 2])

        status.zero_()
        w = torch.zeros(2, H, 112, device="cuda")
        kv.attend(cache, q, d_bad, d_lens, status, weights=w)
        assert int(status) == E_RANGE and (w[0, :, 32:48] == 0).all()
        got = w.cpu().double().numpy()
        for b in range(2):
            tol = r["wslack"][b] * 1.1 + 2.0 ** -15 * r["weights"][b] + 1e-9
            assert (np.abs(got[b, :, :lens[b]] - r["weights"][b]) <= tol).all()

        status.zero_()
        sel = kv.select_pages(cache, q, d_bad, d_lens, 3, status, first=0)
        assert int(status) == E_RANGE and not (sel[0] == 2).any() and (sel >= 0).all()

        status.zero_()
        before = cache.pages.clone()
        k = torch.ones(4, H, D, device="cuda", dtype=torch.float16)
        tail = bad.copy()
        tail[0, 6], tail[0, 2] = wrong, table[0, 2]
        kv.store(cache, k, k, dev(torch, tail), d_lens, status)
        torch.cuda.synchronize()
        assert int(status) == E_RANGE
        touched = (before != cache.pages).any(1).nonzero().flatten().tolist()
        assert touched == [int(table[1, 3])]

        status.zero_()
        cache.pages.copy_(before)
        to = kv.PageCache(torch.zeros(8, kv.page_bytes(T, H, D), dtype=torch.uint8, device="cuda"), T, H, D)
        to_table = np.array([[0, 1, 2], [3, wrong, 5]], np.int32)
        kept, _, _ = kv.evict(cache, d_bad, d_lens, torch.ones(2, H, 100, device="cuda"), 40, to, dev(torch, to_table), status)
        torch.cuda.synchronize()
        assert int(status) == E_RANGE and int(to.pages[[4, 6, 7]].sum()) == 0
        codes = to.codes()[0].float()
        assert (codes[2, :, :8] == 0).all() and not (codes[5, :, :8] == 0).all()     # tokens 32..39 lay in the bad page


def test_bad_lengths_and_starts(fl):
    core, kv, torch = fl
    T, H, G, D, lens = 16, 1, 2, 64, [48, 30]
    rng = np.random.default_rng(4)
    cache, c, table = make(fl, rng, lens, T, H, D)
    q = dev(torch, rng.standard_normal((2, H * G, D)), torch.float32).to(torch.bfloat16)
    for n0, cut in ((49, 48), (2 ** 31 - 1, 48), (-1, 0), (-2 ** 31, 0)):
        status = core.new_status()
        d_lens = dev(torch, np.array([n0, 30], np.int32))
        out = kv.attend(cache, q, dev(torch, table), d_lens, status)
        torch.cuda.synchronize()
        assert int(status) == E_RANGE
        r = ref.attend(c, q.cpu().double().numpy(), table, [cut, 30], [0, 1, 2], 1 / np.sqrt(D))
        check_out(torch, out, None, r, torch.bfloat16, lens, [0, 1, 2])
        before = cache.pages.clone()
        status.zero_()
        k = torch.ones(2, H, D, device="cuda", dtype=torch.float32)
        if n0 > 0:
            kv.store(cache, k, k, dev(torch, table), dev(torch, np.array([n0, 30], np.int32)), status)
            torch.cuda.synchronize()
            touched = (before != cache.pages).any(1).nonzero().flatten().tolist()
            assert int(status) == E_RANGE and touched == [int(table[1, 1])]
            cache.pages.copy_(before)
    for starts in ([0, 3, 2], [-1, 1, 2], [0, 1, 5], [0, 2 ** 31 - 1, 2]):
        status = core.new_status()
        out = torch.full_like(q, 7.0)
        kv.attend(cache, q, dev(torch, table), dev(torch, np.array(lens, np.int32)), status, starts=dev(torch, np.array(starts, np.int32)), out=out)
        sel = kv.select_pages(cache, q, dev(torch, table), dev(torch, np.array(lens, np.int32)), 2, status, starts=dev(torch, np.array(starts, np.int32)))
        torch.cuda.synchronize()
        assert int(status) == E_RANGE


def test_selected_pages_that_are_not_there(fl):
    core, kv, torch = fl
    T, H, G, D, lens = 16, 1, 2, 64, [100]
    rng = np.random.default_rng(4)
    cache, c, table = make(fl, rng, lens, T, H, D)
    q = dev(torch, rng.standard_normal((1, H * G, D)), torch.float32).to(torch.bfloat16)
    sel = np.array([[[3, -1, 2 ** 31 - 1, 900, 6, -5]]], np.int32)
    out = kv.attend(cache, q, torch.nn.functional.pad(dev(torch, table), (0, 3), value=-1), dev(torch, np.array(lens, np.int32)), core.new_status(), selected=dev(torch, sel))
    r = ref.attend(c, q.cpu().double().numpy(), table, lens, [0, 1], 1 / np.sqrt(D), selected=np.array([[[3, 6]]]))
    check_out(torch, out, None, r, torch.bfloat16, lens, [0, 1])
    none = kv.attend(cache, q, dev(torch, table), dev(torch, np.array(lens, np.int32)), core.new_status(), selected=dev(torch, np.full((1, 1, 4), -1, np.int32)))
    assert (none == 0).all()


# ---- together -------------------------------------------------------------------------------------------------------
def move(fl, src, dst, n_pages, order_src, order_dst):
    """Pages of one pool into pages of another, through lane windows, as the transfer path moves them."""
    core, kv, torch = fl
    pb = src.shape[1]
    total = n_pages * pb
    credits, chunk = [3, 1, 2, 2], pb
    tile = next(t for t in range(32768, 0, -128) if pb % t == 0)
    u = core.uniform_params(total, chunk, credits, tile_bytes=tile)
    wins = [torch.empty(total, dtype=torch.uint8, device="cuda") for _ in credits]
    win = core.windows_from_tensors(wins)
    status = core.new_status()
    core.gather_pages_uniform(src, order_src, pb, win, u, status)
    core.scatter_pages_uniform(dst, order_dst, pb, win, u, status)
    torch.cuda.synchronize()
    assert int(status) == 0


def test_prefill_transfer_decode_evict(fl):
    """A prompt is stored and attended to in chunks on one side, its pages travel through lane windows, the other side
    decodes over them, keeps account of the attention, evicts, and goes on over what is left, densely and sparsely."""
    core, kv, torch = fl
    T, H, G, D, B = 16, 2, 4, 128, 2
    rng = np.random.default_rng(11)
    prompts, steps = [150, 83], 6
    total = [p + steps for p in prompts]
    table, n = tables(rng, total, T)
    d_table = dev(torch, table)
    pb = kv.page_bytes(T, H, D)
    left = kv.PageCache(torch.zeros(n, pb, dtype=torch.uint8, device="cuda"), T, H, D)
    status = core.new_status()
    exp = ref.empty(n, T, H, D)
    lens = [0, 0]
    d_lens = torch.zeros(B, dtype=torch.int32, device="cuda")

    def step(cache, exp, table, d_table, d_lens, lens, news, **kw):
        starts = np.concatenate([[0], np.cumsum(news)])
        d_starts = dev(torch, starts.astype(np.int32))
        x = [dev(torch, rng.standard_normal((int(starts[-1]), h, D)), torch.float32).to(torch.bfloat16) for h in (H, H, H * G)]
        kv.store(cache, x[0], x[1], d_table, d_lens, status, starts=d_starts)
        ref.store(exp, x[0].cpu().double().numpy(), x[1].cpu().double().numpy(), table, lens, starts)
        d_lens += dev(torch, np.array(news, np.int32))
        lens = [a + b for a, b in zip(lens, news)]
        out = kv.attend(cache, x[2], d_table, d_lens, status, starts=d_starts, **kw)
        torch.cuda.synchronize()
        r = ref.attend(exp, x[2].cpu().double().numpy(), table, lens, starts, 1 / np.sqrt(D))
        check_out(torch, out, None, r, torch.bfloat16, lens, starts)
        return lens, r

    for news in ([64, 0], [86, 83]):
        lens, _ = step(left, exp, table, d_table, d_lens, lens, news)
    assert lens == prompts
    same_cache(held(left, T, H, D), exp)

    order = np.concatenate([table[b, :-(-lens[b] // T)] for b in range(B)]).astype(np.int32)
    right_order = rng.permutation(n).astype(np.int32)[:len(order)]
    right = kv.PageCache(torch.zeros(n + 9, pb, dtype=torch.uint8, device="cuda"), T, H, D)
    move(fl, left.pages, right.pages, len(order), dev(torch, order), dev(torch, right_order))
    rest = [p for p in range(n + 9) if p not in set(right_order.tolist())]
    table_r, at = np.full_like(table, -1), 0
    for b in range(B):
        m = -(-lens[b] // T)
        table_r[b, :m] = right_order[at:at + m]
        at += m
        for j in range(m, -(-total[b] // T)):
            table_r[b, j] = rest.pop()
    got = held(right, T, H, D)
    for b in range(B):
        for j in range(-(-lens[b] // T)):
            for name in ("k", "v", "s", "low", "high"):
                np.testing.assert_array_equal(got[name][table_r[b, j]], exp[name][table[b, j]])
    exp_r = held(right, T, H, D)
    d_table_r = dev(torch, table_r)
    weights = torch.zeros(B, H, max(total), device="cuda")
    sums = np.zeros((B, H, max(total)))
    for _ in range(steps):
        lens, r = step(right, exp_r, table_r, d_table_r, d_lens, lens, [1, 1], weights=weights)
        for b in range(B):
            sums[b, :, :lens[b]] += r["weights"][b]
    assert np.abs(weights.cpu().double().numpy() - sums).max() <= steps * G * 2.0 ** -15

    budget = 64
    per = budget // T + 1
    to = kv.PageCache(torch.zeros(per * B, pb, dtype=torch.uint8, device="cuda"), T, H, D)
    table_t = np.arange(per * B, dtype=np.int32).reshape(B, per)
    w = weights.cpu().numpy()
    kept, new_w, d_lens = kv.evict(right, d_table_r, d_lens, weights, budget, to, dev(torch, table_t), status, first=2, recent=8)
    exp_t = ref.empty(per * B, T, H, D)
    k, _ = ref.evict(exp_r, table_r, lens, w, budget, 2, 8, exp_t, table_t)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(kept.cpu().numpy(), k)
    same_cache(held(to, T, H, D), exp_t)
    lens = [min(x, budget) for x in lens]
    lens, _ = step(to, exp_t, table_t, dev(torch, table_t), d_lens, lens, [1, 1])
    q = dev(torch, rng.standard_normal((B, H * G, D)), torch.float32).to(torch.bfloat16)
    sel = kv.select_pages(to, q, dev(torch, table_t), d_lens, 3, status)
    out = kv.attend(to, q, dev(torch, table_t), d_lens, status, selected=sel)
    torch.cuda.synchronize()
    exp_sel = ref.select(exp_t, q.cpu().double().numpy(), table_t, lens, [0, 1, 2], 3, 1, 1)
    np.testing.assert_array_equal(sel.cpu().numpy(), exp_sel)
    check_out(torch, out, None, ref.attend(exp_t, q.cpu().double().numpy(), table_t, lens, [0, 1, 2], 1 / np.sqrt(D), selected=exp_sel), torch.bfloat16, lens, [0, 1, 2])
    assert int(status) == 0


# ---- graphs and streams ---------------------------------------------------------------------------------------------
def decode_step(kv, s):
    kv.store(s["cache"], s["k"], s["v"], s["table"], s["lens"], s["status"])
    s["lens"] += 1
    s["out"] = kv.attend(s["cache"], s["q"], s["table"], s["lens"], s["status"], weights=s["w"])
    s["sel"] = kv.select_pages(s["cache"], s["q"], s["table"], s["lens"], 5, s["status"])
    s["sparse"] = kv.attend(s["cache"], s["q"], s["table"], s["lens"], s["status"], selected=s["sel"])
    s["kept"], s["nw"], s["nl"] = kv.evict(s["cache"], s["table"], s["lens"], s["w"], 40, s["to"], s["to_table"], s["status"], first=1, recent=4)
    return [s[x].clone() for x in ("out", "sel", "sparse", "kept", "nw", "nl", "w")] + [s["cache"].pages.clone(), s["to"].pages.clone()]


def decode_state(fl, rng, B=3):
    core, kv, torch = fl
    T, H, G, D = 16, 2, 4, 64
    lens = [200, 55, 16][:B]
    table, n = tables(rng, [x + 64 for x in lens], T)
    cache = kv.PageCache(torch.zeros(n, kv.page_bytes(T, H, D), dtype=torch.uint8, device="cuda"), T, H, D)
    total = sum(lens)
    k, v = (dev(torch, rng.standard_normal((total, H, D)), torch.float32) for _ in range(2))
    status = core.new_status()
    starts = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    kv.store(cache, k, v, dev(torch, table), torch.zeros(B, dtype=torch.int32, device="cuda"), status, starts=dev(torch, starts))
    to = kv.PageCache(torch.zeros(3 * B, kv.page_bytes(T, H, D), dtype=torch.uint8, device="cuda"), T, H, D)
    f = lambda h: dev(torch, rng.standard_normal((B, h, D)), torch.float32).to(torch.bfloat16)
    return dict(cache=cache, table=dev(torch, table), lens=dev(torch, np.array(lens, np.int32)), k=f(H), v=f(H), q=f(H * G), status=status,
                w=torch.zeros(B, H, 300, device="cuda"), to=to, to_table=torch.arange(3 * B, dtype=torch.int32, device="cuda").view(B, 3))


def test_graph_replays_equal_eager_steps(fl):
    """Two graphs of a decode step with new inputs before every replay, eager work of the same kind between them."""
    core, kv, torch = fl
    a = [decode_state(fl, np.random.default_rng(s)) for s in (1, 2)]
    e = [decode_state(fl, np.random.default_rng(s)) for s in (1, 2)]
    side = torch.cuda.Stream()
    graphs = []
    for s in a:
        keep = {x: s[x].clone() for x in ("lens", "w")}
        pages, to = s["cache"].pages.clone(), s["to"].pages.clone()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            decode_step(kv, s)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s["res"] = decode_step(kv, s)
        for x, y in keep.items():
            s[x].copy_(y)
        s["cache"].pages.copy_(pages)
        s["to"].pages.copy_(to)
        graphs.append(g)
    rng = np.random.default_rng(3)
    for turn in range(5):
        for i in (0, 1):
            for name in ("k", "v", "q"):
                x = dev(torch, rng.standard_normal(tuple(a[i][name].shape)), torch.float32).to(torch.bfloat16)
                a[i][name].copy_(x)
                e[i][name].copy_(x)
            graphs[i].replay()
            exp = decode_step(kv, e[i])
            if turn % 2:
                torch.cuda.synchronize()
            for x, y in zip(a[i]["res"], exp):
                assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    assert int(a[0]["status"]) == int(a[1]["status"]) == 0


def test_results_do_not_depend_on_the_run_or_the_stream(fl):
    """The same calls on two other streams at once, the inputs dropped right after them: the same bits."""
    core, kv, torch = fl
    exp = [decode_step(kv, decode_state(fl, np.random.default_rng(s))) for s in (5, 6)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(3):
        got = []
        for s, st in zip((5, 6), streams):
            x = decode_state(fl, np.random.default_rng(s))
            q = [x["q"].clone() for _ in range(3)]                 # dropped one by one; made before the streams meet
            st.wait_stream(torch.cuda.current_stream())
            kw = dict(stream=st)
            kv.store(x["cache"], x["k"], x["v"], x["table"], x["lens"], x["status"], **kw)
            with torch.cuda.stream(st):
                x["lens"] += 1
            out = kv.attend(x["cache"], q.pop(), x["table"], x["lens"], x["status"], weights=x["w"], **kw)
            sel = kv.select_pages(x["cache"], q.pop(), x["table"], x["lens"], 5, x["status"], **kw)
            sparse = kv.attend(x["cache"], q.pop(), x["table"], x["lens"], x["status"], selected=sel, **kw)
            kept, nw, nl = kv.evict(x["cache"], x["table"], x["lens"], x["w"], 40, x["to"], x["to_table"], x["status"], first=1, recent=4, **kw)
            got.append([out, sel, sparse, kept, nw, nl, x["w"], x["cache"].pages, x["to"].pages])
            del x
            junk = [torch.full((3, 8, 64), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(50)]
        torch.cuda.synchronize()
        for g, e in zip(got, exp):
            for x, y in zip(g, e):
                assert torch.equal(x.contiguous().view(torch.uint8), y.view(torch.uint8))


def test_empty_calls(fl):
    core, kv, torch = fl
    T, H, G, D = 16, 1, 2, 64
    rng = np.random.default_rng(0)
    cache, c, table = make(fl, rng, [20, 30], T, H, D)
    status = core.new_status()
    none = torch.empty(0, H, D, dtype=torch.bfloat16, device="cuda")
    d_table, lens = dev(torch, table), dev(torch, np.array([20, 30], np.int32))
    before = cache.pages.clone()
    kv.store(cache, none, none, d_table, lens, status)
    q = torch.empty(0, H * G, D, dtype=torch.bfloat16, device="cuda")
    w_in = torch.rand(2, H, 40, device="cuda")
    w = torch.zeros_like(w_in)
    assert kv.attend(cache, q, d_table, lens, status, weights=w, weights_in=w_in).shape == q.shape
    assert kv.select_pages(cache, q, d_table, lens, 3, status).shape == (0, H, 3)
    assert kv.attend(cache, q, d_table, lens, status, selected=torch.empty(0, H, 2, dtype=torch.int32, device="cuda")).shape == q.shape
    torch.cuda.synchronize()
    assert torch.equal(w, w_in) and torch.equal(before, cache.pages) and int(status) == 0


# ---- pages that are not there ---------------------------------------------------------------------------------------
WORDS = [-0x55555556, 0x5D800000, 0x7F800000, 0x7FC00000]        # scale words of pages that hold nothing: 0xAAAAAAAA, 2^60, infinity, NaN


def strewn(fl, cache, table, word):
    """The same pool behind a page that no table names, every scale word of a page that holds nothing being `word`: (cache, table, an idle page)."""
    core, kv, torch = fl
    c = kv.PageCache(torch.cat([torch.full_like(cache.pages[:1], 0xAA), cache.pages]), cache.tokens, cache.heads, cache.dim)
    used = set((table[table >= 0] + 1).tolist())
    idle = [p for p in range(c.pages.shape[0]) if p not in used]
    c.scales().view(torch.int32)[idle] = word
    return c, np.where(table < 0, table, table + 1).astype(np.int32), idle[-1]


@pytest.mark.parametrize("T", [16, 48])
@pytest.mark.parametrize("n,H,G", [(1, 2, 4), (5, 2, 4), (20, 2, 4), (40, 65, 4)])
@pytest.mark.parametrize("word", WORDS, ids=hex)
def test_absent_page_is_not_seen(fl, T, n, H, G, word):
    """Whatever lies in the pool's first page, a page number outside the pool only takes its own keys away."""
    core, kv, torch = fl
    D, lens = 64, [7 * T - 5, 4 * T]
    rng = np.random.default_rng(T + n)
    cache, c, table = make(fl, rng, lens, T, H, D)
    cache, moved, _ = strewn(fl, cache, table, word)
    moved[0, 2] = -1
    q = dev(torch, rng.standard_normal((2 * n, H * G, D)), torch.float32).to(torch.bfloat16)
    status, w = core.new_status(), torch.zeros(2, H, 7 * T, device="cuda")
    lse = torch.zeros(2 * n, H * G, device="cuda")
    out = kv.attend(cache, q, dev(torch, moved), dev(torch, np.array(lens, np.int32)), status, weights=w, lse=lse)
    assert int(status) == E_RANGE
    pick = np.full((2 * n, H, 7), -1)
    pick[:n, :, :6], pick[n:, :, :4] = [0, 1, 3, 4, 5, 6], range(4)
    starts = [0, n, 2 * n]
    r = ref.attend(c, q.cpu().double().numpy(), table, lens, starts, 1 / np.sqrt(D), selected=pick)
    check_out(torch, out, lse, r, torch.bfloat16, lens, starts)
    for b, x in enumerate(lens):
        tol = r["wslack"][b] * 1.1 + r["weights"][b] * (n * G + 64) * 2.0 ** -23
        assert (np.abs(w[b, :, :x].cpu().double().numpy() - r["weights"][b]) <= tol).all()


@pytest.mark.parametrize("T", [16, 48])
@pytest.mark.parametrize("G", [2, 20])
@pytest.mark.parametrize("word", WORDS, ids=hex)
def test_selected_index_behind_the_sequence_is_not_seen(fl, T, G, word):
    """Indices behind the sequence's pages, where the table names no page or one that nothing was stored in: no error, no keys."""
    core, kv, torch = fl
    H, D, lens = 2, 64, [7 * T - 5]
    rng = np.random.default_rng(T + G)
    cache, c, table = make(fl, rng, lens, T, H, D)
    cache, moved, idle = strewn(fl, cache, table, word)
    moved = np.concatenate([moved, np.array([[-1, idle, -1]], np.int32)], 1)
    q = dev(torch, rng.standard_normal((1, H * G, D)), torch.float32).to(torch.bfloat16)
    for sel, seen in (([3, 7, 6, 1], [1, 3, 6]), ([3, 8, 6, 0, 9], [0, 3, 6]), ([8, 5], [5]), ([9, 8, 7, 2], [2])):
        d_sel = dev(torch, np.broadcast_to(np.array(sel, np.int32), (1, H, len(sel))))
        status = core.new_status()
        out = kv.attend(cache, q, dev(torch, moved), dev(torch, np.array(lens, np.int32)), status, selected=d_sel)
        assert int(status) == 0
        r = ref.attend(c, q.cpu().double().numpy(), table, lens, [0, 1], 1 / np.sqrt(D), selected=np.broadcast_to(np.array(seen), (1, H, len(seen))))
        check_out(torch, out, None, r, torch.bfloat16, lens, [0, 1])


def test_evict_does_not_write_the_lengths_it_reads(fl):
    core, kv, torch = fl
    T, H, D, x = 16, 2, 64, 40
    cache, c, table = make(fl, np.random.default_rng(2), [x, x], T, H, D)
    words = dev(torch, np.array([x, x, 0, 0], np.int32))
    to = kv.PageCache(torch.zeros(4, kv.page_bytes(T, H, D), dtype=torch.uint8, device="cuda"), T, H, D)
    args = torch.ones(2, H, x, device="cuda"), 20, to, dev(torch, np.arange(4, dtype=np.int32).reshape(2, 2)), core.new_status()
    for new_lens in (words[:2], words[1:3]):
        with pytest.raises(ValueError, match="new_lens overlaps lens"):
            kv.evict(cache, dev(torch, table), words[:2], *args, new_lens=new_lens)
    kv.evict(cache, dev(torch, table), words[:2], *args, new_lens=words[2:])
    assert words.tolist() == [x, x, 20, 20] and int(args[-1]) == 0


def test_evict_does_not_pack_into_the_pages_it_reads(fl):
    core, kv, torch = fl
    T, H, D, x = 16, 2, 64, 40
    cache, c, table = make(fl, np.random.default_rng(2), [x, x], T, H, D)
    d_table, lens, status = dev(torch, table), dev(torch, np.array([x, x], np.int32)), core.new_status()
    w, before = torch.ones(2, H, x, device="cuda"), cache.pages.clone()
    with pytest.raises(ValueError, match="new pages"):
        kv.evict(cache, d_table, lens, w, 20, cache, d_table, status)
    other = kv.PageCache(torch.zeros_like(cache.pages), T, H, D)
    kv.evict(cache, d_table, lens, w, 20, other, d_table, status)            # the same numbers in another pool are other pages
    assert int(status) == 0 and torch.equal(before, cache.pages) and int(other.pages[int(table[0, 0])].sum()) > 0


def test_refused_calls_leave_the_stream_alone(fl):
    """What is refused on a named stream is refused as elsewhere, and the caller's stream stays the current one."""
    core, kv, torch = fl
    T, H, G, D, x = 16, 2, 4, 64, 40
    rng = np.random.default_rng(2)
    cache, c, table = make(fl, rng, [x, x], T, H, D)
    q = dev(torch, rng.standard_normal((2, H * G, D)), torch.float32).to(torch.bfloat16)
    d_table, lens, status = dev(torch, table), dev(torch, np.array([x, x], np.int32)), core.new_status()
    w = torch.ones(2, H, 64, device="cuda")
    to = kv.PageCache(torch.zeros(4, kv.page_bytes(T, H, D), dtype=torch.uint8, device="cuda"), T, H, D)
    to_table = dev(torch, np.arange(4, dtype=np.int32).reshape(2, 2))
    side, here = torch.cuda.Stream(), torch.cuda.current_stream()
    host = lambda dtype, *shape: torch.zeros(*shape, dtype=dtype)
    evict = lambda **kw: kv.evict(cache, d_table, lens, w, 20, to, to_table, status, **kw)
    calls = [lambda **kw: kv.attend(cache, q, d_table, lens, status, out=q.cpu(), **kw),
             lambda **kw: kv.attend(cache, q, d_table, lens, status, weights=w, workspace=host(torch.uint8, 1 << 20), **kw),
             lambda **kw: kv.select_pages(cache, q, d_table, lens, 2, status, out=host(torch.int32, 2, H, 2), **kw),
             lambda **kw: kv.select_pages(cache, q, d_table, lens, 2, status, workspace=host(torch.uint8, 1 << 20), **kw),
             lambda **kw: evict(kept=host(torch.int32, 2, H, 20), **kw), lambda **kw: evict(new_weights=host(torch.float32, 2, H, 20), **kw),
             lambda **kw: evict(new_lens=host(torch.int32, 2), **kw)]
    for call in calls:
        for kw in ({}, dict(stream=side)):
            with pytest.raises(ValueError):
                call(**kw)
            assert torch.cuda.current_stream() == here
    assert int(status) == 0


@pytest.mark.parametrize("n0", [-1, -2 ** 31])
def test_store_skips_a_sequence_of_negative_length(fl, n0):
    """Nothing of such a sequence is written, above all not its first tokens; the others' tokens are stored."""
    core, kv, torch = fl
    T, H, D = 16, 2, 64
    rng = np.random.default_rng(4)
    cache, c, table = make(fl, rng, [48, 30, 17], T, H, D)
    exp = held(cache, T, H, D)
    k, v = (dev(torch, rng.standard_normal((6, H, D)), torch.float32) for _ in range(2))
    status = core.new_status()
    kv.store(cache, k, v, dev(torch, table), dev(torch, np.array([n0, 30, 17], np.int32)), status)
    assert int(status) == E_RANGE
    ref.store(exp, k.cpu().double().numpy(), v.cpu().double().numpy(), table, [48, 30, 17], [2, 2, 4, 6])
    same_cache(held(cache, T, H, D), exp)


STARTS = [[0, 3, 2], [-1, 1, 2], [0, 1, 5], [0, 2 ** 31 - 1, 2], [0, -2 ** 31, 2], [0, 2, 9, 3], [1, 3, -1, 4], [5, 5, 6, 4]]


@pytest.mark.parametrize("starts", STARTS, ids=str)
@pytest.mark.parametrize("H,G", [(1, 2), (33, 210)])
def test_bad_starts(fl, starts, H, G):
    """Each entry point reports starts that leave the call's tokens or descend, skips those sequences and serves the others."""
    core, kv, torch = fl
    T, D = 16, 32
    B, lens = len(starts) - 1, [48, 30, 20][:len(starts) - 1]
    n = 2 if B == 2 else 4
    rng = np.random.default_rng(4)
    cache, c, table = make(fl, rng, lens, T, H, D)
    ok = [0 <= a <= b <= n for a, b in zip(starts, starts[1:])]
    news = [b - a if o else 0 for a, b, o in zip(starts, starts[1:], ok)]
    tok = [range(a, b) if o else range(0) for a, b, o in zip(starts, starts[1:], ok)]
    order = [i for t in tok for i in t]                       # the tokens that are somebody's, sequence by sequence
    packed = np.concatenate([[0], np.cumsum(news)])
    d_table, d_lens, d_starts = dev(torch, table), dev(torch, np.array(lens, np.int32)), dev(torch, np.array(starts, np.int32))
    q = dev(torch, rng.standard_normal((n, H * G, D)), torch.float32).to(torch.bfloat16)
    qn = q.cpu().double().numpy()[order]
    nobody = [i for i in range(n) if i not in order]

    status, w_in = core.new_status(), torch.rand(B, H, 50, device="cuda")
    out, lse, w = torch.full_like(q, 7.0), torch.full((n, H * G), 7.0, device="cuda"), torch.full_like(w_in, -1.0)
    kv.attend(cache, q, d_table, d_lens, status, starts=d_starts, out=out, lse=lse, weights=w, weights_in=w_in)
    assert int(status) == E_RANGE and (out[nobody] == 7).all() and (lse[nobody] == 7).all()
    r = ref.attend(c, qn, table, lens, packed, 1 / np.sqrt(D))
    check_out(torch, out[order], lse[order], r, torch.bfloat16, lens, packed)
    got, base = (x.cpu().double().numpy() for x in (w, w_in))
    for b, x in enumerate(lens):
        tol = r["wslack"][b] * 1.1 + (r["weights"][b] + base[b, :, :x]) * (n * G + 64) * 2.0 ** -23
        assert (np.abs(got[b, :, :x] - base[b, :, :x] - r["weights"][b]) <= tol).all()
        np.testing.assert_array_equal(got[b, :, x:], base[b, :, x:])

    status.zero_()
    sel = torch.full((n, H, 2), -7, dtype=torch.int32, device="cuda")
    kv.select_pages(cache, q, d_table, d_lens, 2, status, starts=d_starts, out=sel)
    assert int(status) == E_RANGE and (sel[nobody] == -7).all()
    exp = ref.select(c, qn, table, lens, packed, 2, 1, 1)
    np.testing.assert_array_equal(sel.cpu().numpy()[order], exp)

    status.zero_()
    out.fill_(7.0)
    kv.attend(cache, q, d_table, d_lens, status, starts=d_starts, out=out, selected=sel)
    assert int(status) == E_RANGE and (out[nobody] == 7).all()
    check_out(torch, out[order], None, ref.attend(c, qn, table, lens, packed, 1 / np.sqrt(D), selected=exp), torch.bfloat16, lens, packed)

    status.zero_()
    before, c2 = cache.pages.clone(), held(cache, T, H, D)
    k, v = (dev(torch, rng.standard_normal((n, H, D)), torch.float32) for _ in range(2))
    had = [x - 4 for x in lens]
    kv.store(cache, k, v, d_table, dev(torch, np.array(had, np.int32)), status, starts=d_starts)
    assert int(status) == E_RANGE
    ref.store(c2, k.cpu().double().numpy()[order], v.cpu().double().numpy()[order], table, had, packed)
    same_cache(held(cache, T, H, D), c2)
    mine = {int(table[b, p // T]) for b in range(B) for p in range(had[b], had[b] + news[b])}
    assert set((before != cache.pages).any(1).nonzero().flatten().tolist()) <= mine


@pytest.mark.parametrize("size", [1e38, 1e-35, 1e-36])
@pytest.mark.parametrize("n,x,H,G,D", [(1, 50, 2, 4, 64), (1, 9000, 1, 2, 64), (20, 200, 2, 4, 128), (20, 1500, 2, 4, 128), (3, 300, 1, 2, 256), (40, 90, 65, 4, 128), (40, 600, 65, 4, 128),
                                       (100, 400, 1, 4, 256)])
def test_attend_values_near_the_ends_of_the_range(fl, size, n, x, H, G, D):
    """Outputs are averages of the values: where those are representable, so are these, whatever the sums pass on the way."""
    core, kv, torch = fl
    T = 16
    rng = np.random.default_rng(n + x)
    k, v = rng.standard_normal((x, H, D)), rng.uniform(0.5, 2, (x, H, D)) * size
    table, pages = tables(rng, [x], T)
    c = ref.empty(pages, T, H, D)
    ref.store(c, k, v, table, [0], [0, x])
    cache = records(fl, c, T, H, D, [x], table)
    q = dev(torch, rng.standard_normal((n, H * G, D)), torch.float32).to(torch.bfloat16)
    status = core.new_status()
    out = kv.attend(cache, q, dev(torch, table), dev(torch, np.array([x], np.int32)), status).cpu().double().numpy()
    r = ref.attend(c, q.cpu().double().numpy(), table, [x], [0, n], 1 / np.sqrt(D))
    # all values are within a factor of 4 of each other: no probability is lost beside another; 2^-140: 256 parts of 2^-149 and less
    tol = ref.out_tolerance(r, torch.finfo(torch.bfloat16).eps, x) - 1e-30 + 2.0 ** -140
    assert int(status) == 0 and (np.abs(out - r["out"]) <= tol).all()


@pytest.mark.parametrize("T2", [16, 32])
def test_evict_by_weights_of_fewer_positions(fl, T2):
    """Sequences longer than their weights are cut off there: what is packed, counted and bounded is what the weights know."""
    core, kv, torch = fl
    T, H, D, lens, width, budget = 16, 2, 64, [100, 60, 20], 41, 50
    rng = np.random.default_rng(6)
    cache, c, table = make(fl, rng, lens, T, H, D)
    w = rng.random((3, H, width)).astype(np.float32)
    per = -(-budget // T2)
    table2 = np.arange(3 * per, dtype=np.int32).reshape(3, per)
    to = kv.PageCache(torch.full((3 * per, kv.page_bytes(T2, H, D)), 0xA5, dtype=torch.uint8, device="cuda"), T2, H, D)
    exp = held(to, T2, H, D)
    status = core.new_status()
    kept, nw, nl = kv.evict(cache, dev(torch, table), dev(torch, np.array(lens, np.int32)), dev(torch, w), budget, to, dev(torch, table2), status)
    assert int(status) == E_RANGE
    cut = [min(x, width) for x in lens]
    k, x = ref.evict(c, table, cut, w, budget, 0, 0, exp, table2)
    np.testing.assert_array_equal(nl.cpu().numpy(), cut)
    np.testing.assert_array_equal(kept.cpu().numpy(), k)
    same_numbers(nw.cpu().double().numpy(), x, "weights")
    same_cache(held(to, T2, H, D), exp)


def test_parameters_without_recording(fl):
    """Keys, values and queries made of parameters: served where no gradient is recorded, as detached ones are."""
    core, kv, torch = fl
    T, H, G, D, x = 16, 2, 4, 64, 40
    cache, c, table = make(fl, np.random.default_rng(2), [x], T, H, D)
    args = dev(torch, table), dev(torch, np.array([x], np.int32)), core.new_status()
    w = torch.randn(D, H * G * D, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    q = (torch.randn(1, D, device="cuda", dtype=torch.bfloat16) @ w).view(1, H * G, D)
    with pytest.raises(ValueError, match="no gradient"):
        kv.attend(cache, q, *args)
    exp = kv.attend(cache, q.detach(), *args)
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            assert torch.equal(kv.attend(cache, q, *args), exp)


@pytest.mark.parametrize("gap", [6, 7, 12, 24, 40, 60])
@pytest.mark.parametrize("n,H,G,D", [(20, 1, 1, 64), (40, 2, 1, 128), (64, 1, 4, 64), (64, 66, 4, 128), (64, 1, 4, 256), (64, 2, 1, 256)])
def test_attend_value_scales_apart_from_page_to_page(fl, gap, n, H, G, D):
    """Neighbouring pages whose value scales are 2^gap apart: queries that see only the smaller ones, and queries to whom the larger ones'
    keys are worth nothing, get their averages as exactly as without such neighbours."""
    core, kv, torch = fl
    T, x = 16, 64
    rng = np.random.default_rng(gap + n)
    k, v = rng.standard_normal((x, H, D)), rng.uniform(0.5, 1, (x, H, D)) * 2.0 ** -(gap // 2)
    for j in (1, 2):
        v[j * T:(j + 1) * T] *= 2.0 ** gap
        k[j * T:(j + 1) * T, :, 0] = -150.0                      # times a query of 8 or 0 there, over sqrt(D): worth nothing, or as much as others
    k[:T, :, 0] = k[3 * T:, :, 0] = 0
    table, pages = tables(rng, [x], T)
    c = ref.empty(pages, T, H, D)
    ref.store(c, k, v, table, [0], [0, x])
    cache = records(fl, c, T, H, D, [x], table)
    qn = rng.standard_normal((n, H * G, D))
    qn[:, :, 0] = np.where(np.arange(n)[:, None] % 3 == 0, 12.0, 0.0)
    q = dev(torch, qn, torch.float32).to(torch.bfloat16)
    status = core.new_status()
    for causal in (True, False):
        out = kv.attend(cache, q, dev(torch, table), dev(torch, np.array([x], np.int32)), status, causal=causal).cpu().double().numpy()
        r = ref.attend(c, q.cpu().double().numpy(), table, [x], [0, n], 1 / np.sqrt(D), causal)
        tol = ref.out_tolerance(r, torch.finfo(torch.bfloat16).eps, x) - 1e-30 + 2.0 ** -140
        assert int(status) == 0 and (np.abs(out - r["out"]) <= tol).all()


@pytest.mark.parametrize("at", [3, 21, 50])
@pytest.mark.parametrize("n,H,G,D", [(1, 2, 4, 64), (20, 1, 4, 128), (64, 1, 4, 64), (64, 66, 4, 128), (64, 1, 4, 256)])
def test_attend_nan_beside_value_scales_apart(fl, at, n, H, G, D):
    """A NaN among the values of a page that is taken apart from its neighbour reaches those that see it, and no other."""
    core, kv, torch = fl
    T, x = 16, 64
    rng = np.random.default_rng(n)
    k, v = rng.standard_normal((x, H, D)), rng.uniform(0.5, 1, (x, H, D))
    v[T:3 * T] *= 2.0 ** 24
    table, pages = tables(rng, [x], T)
    c = ref.empty(pages, T, H, D)
    ref.store(c, k, v, table, [0], [0, x])
    c["v"][table[0, at // T], H - 1, at % T, 5] = np.nan
    cache = records(fl, c, T, H, D, [x], table)
    q = dev(torch, rng.standard_normal((n, H * G, D)), torch.float32).to(torch.bfloat16)
    for causal in (True, False):
        out = kv.attend(cache, q, dev(torch, table), dev(torch, np.array([x], np.int32)), core.new_status(), causal=causal).cpu().double().numpy()
        with np.errstate(invalid="ignore"):
            r = ref.attend(c, q.cpu().double().numpy(), table, [x], [0, n], 1 / np.sqrt(D), causal)
        nan = np.isnan(r["out"])
        seen = (x - n + 1 + np.arange(n) > at) if causal else np.ones(n, bool)
        assert (nan[:, (H - 1) * G:, 5].all(1) == seen).all() and nan.sum() == seen.sum() * G
        np.testing.assert_array_equal(np.isnan(out), nan)
        assert (np.abs(out - r["out"]) <= ref.out_tolerance(r, torch.finfo(torch.bfloat16).eps, x))[~nan].all()


@pytest.mark.parametrize("n,x,H,G", [(1, 50, 2, 4), (20, 200, 2, 4), (40, 90, 65, 4)])
def test_attend_least_keys_under_huge_queries(fl, n, x, H, G):
    """Keys at the least scale there is, under queries as large as their products with the codes allow: the scores are what they are."""
    core, kv, torch = fl
    T, D = 16, 64
    rng = np.random.default_rng(n + x)
    k, v = rng.standard_normal((x, H, D)) * 1e-37, rng.standard_normal((x, H, D))
    table, pages = tables(rng, [x], T)
    c = ref.empty(pages, T, H, D)
    ref.store(c, k, v, table, [0], [0, x])
    assert (c["s"][table[0], :, 0] == 2.0 ** -126).all()
    cache = records(fl, c, T, H, D, [x], table)
    q = dev(torch, rng.standard_normal((n, H * G, D)) * 1e35, torch.float32).to(torch.bfloat16)
    # no order of a sum of |q| |code| passes the range
    assert (np.abs(q.cpu().double().numpy()).max(2) * np.nansum(np.abs(c["k"]), 3).max() < 2.0 ** 128).all()
    status, w, lse = core.new_status(), torch.zeros(1, H, x, device="cuda"), torch.zeros(n, H * G, device="cuda")
    out = kv.attend(cache, q, dev(torch, table), dev(torch, np.array([x], np.int32)), status, scale=1.0, weights=w, lse=lse)
    assert int(status) == 0
    r = ref.attend(c, q.cpu().double().numpy(), table, [x], [0, n], 1.0)
    check_out(torch, out, lse, r, torch.bfloat16, [x], [0, n])
    tol = r["wslack"][0] * 1.1 + r["weights"][0] * (n * G + 64) * 2.0 ** -23
    assert (np.abs(w[0].cpu().double().numpy() - r["weights"][0]) <= tol).all()
