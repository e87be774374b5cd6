"""The paged cache on the GPU (plan, append, attention, and the three in a row) against float64."""
import ctypes as C

import numpy as np
import pytest

import paged_cases as ref
from ruai_b200 import nn

pytestmark = pytest.mark.gpu

RD = {"f32": nn.F32, "f16": nn.F16, "bf16": nn.BF16}
NP = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}


@pytest.fixture(scope="module")
def dev():
    assert nn.Device.is_available(), "these tests need a CUDA device"
    return nn.Device.cuda(0)


def ints(dev, a):
    return nn.Tensor.from_numpy(dev, np.asarray(a, np.int32))


def put(dev, a, dtype):
    """(tensor, the numbers that it holds)"""
    s, n = ref.stored(a, dtype)
    return nn.Tensor.from_numpy(dev, s, RD[dtype]), n


def numbers(t):
    a = t.numpy()
    return ref.from_bf16(a) if t.rdtype == nn.BF16 else a.astype(np.float64)


def lay_out(rng, lens, page, spare=3, extra=1):
    """Pages for requests of these lengths in a random order: (table, pages)."""
    held = [ref.up(int(n), page) for n in lens]
    pages = sum(held) + spare
    order = rng.permutation(pages)
    table, at = np.full((len(lens), max(held + [1]) + extra), -1), 0
    for r, h in enumerate(held):
        table[r, :h] = order[at:at + h]
        at += h
    return table, pages


# ---- plan -----------------------------------------------------------------------------------------------------------------


def run_plan(dev, cached, fresh, table, ring, words, page, tokens, in_place=False):
    t, r, w = ints(dev, table), ints(dev, ring), ints(dev, words)
    out = nn.PagePlan(ints(dev, np.full(len(cached) + 1, 77)), ints(dev, np.full(tokens, 77)), ints(dev, np.full(tokens, 77)), w if in_place else ints(dev, [77, 77, 77]))
    nn.page_plan(ints(dev, cached), ints(dev, fresh), t, r, w, page, out=out)
    return [x.numpy().astype(np.int64) for x in (t, r, out.starts, out.positions, out.slots, out.words)]


@pytest.mark.parametrize("R,tokens,page", [(1, 1, 16), (1, 300, 16), (2, 0, 32), (33, 40, 16), (256, 256, 64), (257, 257, 16), (1000, 3000, 256), (2049, 2049, 16), (2500, 40000, 32), (8192, 9000, 16)])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan(dev, R, tokens, page, in_place):
    rng = np.random.default_rng(R + page)
    cached = np.where(rng.random(R) < 0.2, 0, rng.integers(0, 40 * page if R < 3000 else 2 * page, R))
    cached[::3] = cached[::3] // page * page  # lengths at a page's end
    fresh = np.minimum(1, rng.integers(0, 4, R))
    fresh[rng.random(R) < 0.1] = -1
    while fresh.clip(0).sum() > tokens:
        fresh[rng.integers(R)] = 0
    if tokens > fresh.clip(0).sum():  # one request takes the rest, bar some padding
        r = int(rng.integers(R))
        fresh[r] = max(fresh[r], 0) + (tokens - fresh.clip(0).sum()) * 3 // 4
    table, pages = lay_out(rng, cached, page, spare=int(ref.up(tokens, page)) + R, extra=ref.up(tokens, page) + 1)
    used = set(table[table >= 0].tolist())
    free = rng.permutation([p for p in range(pages) if p not in used])
    first = int(rng.integers(pages))
    ring = np.full(pages, -1)
    ring[(first + np.arange(len(free))) % pages] = free
    words = [first, len(free), 0]
    want = ref.plan(cached, fresh, table, ring, words, page, tokens)
    got = run_plan(dev, cached, fresh, table, ring, words, page, tokens, in_place)
    dev.synchronize()
    for name, a, b in zip(("table", "ring", "starts", "positions", "slots", "words"), want, got):
        assert np.array_equal(a, b), name


@pytest.mark.parametrize("cached,fresh,words,missing", [([16, 3], [1, 40], [0, 2, 0], 1), ([16, -1], [1, 1], [0, 9, 0], 0), ([16, 3], [1, 200], [0, 9, 0], 0), ([2**31 - 1, 3], [1, 1], [0, 9, 0], 0),
                                                        ([100, 3], [-1, 1], [0, 9, 0], 0), ([16, 3], [60, 60], [0, 9, 0], 0), ([16, 3], [1, 1], [10, 2, 0], 0), ([16, 3], [1, 1], [0, 11, 0], 0),
                                                        ([16, 3], [1, 1], [-1, 2, 0], 0), ([64, 3], [-1, 0], [0, 7, 0], 0)])
def test_plan_refuses_on_the_device(dev, cached, fresh, words, missing):
    """Too few pages, lengths outside the table or the step, words outside the ring: nothing is planned, and the host is told."""
    table, ring = np.array([[1, 2, 3, 4], [5, -1, -1, -1]]), np.arange(10)
    with_words = list(words)
    got = run_plan(dev, cached, fresh, table, ring, words, 16, 100)
    with pytest.raises(nn.RuaiError, match="page plan was refused"):
        dev.synchronize()
    dev.synchronize()
    assert np.array_equal(got[0], table) and np.array_equal(got[1], ring) and not got[2].any() and (got[3] == -1).all() and (got[4] == -1).all()
    assert got[5].tolist() == [with_words[0], with_words[1], missing]


def test_plan_page_out_of_range(dev):
    got = run_plan(dev, [3, 20], [1, 1], np.array([[12, -1], [4, -7]]), np.arange(10), [0, 0, 0], 16, 3)
    with pytest.raises(nn.RuaiError, match="out of range"):
        dev.synchronize()
    assert got[3].tolist() == [3, 20, -1] and got[4].tolist() == [-1, -1, -1]


def test_plans_in_a_row_lose_no_page(dev):
    """Requests that grow, end and come again: at every step the pages held and the free ones are all pages, once."""
    rng = np.random.default_rng(5)
    R, page, pages, width = 9, 16, 60, 12
    cached, table, ring, words = np.zeros(R, np.int64), np.full((R, width), -1), rng.permutation(pages), [3, 60, 0]
    for _ in range(40):
        room = np.minimum(width * page - cached, 20)
        fresh = np.where(rng.random(R) < 0.15, -1, rng.integers(0, 20, R)).clip(max=room)
        want = ref.plan(cached, fresh, table, ring, words, page, 200)
        if want is None:
            fresh = np.full(R, -1)
            want = ref.plan(cached, fresh, table, ring, words, page, 200)
        got = run_plan(dev, cached, fresh, table, ring, words, page, 200)
        for a, b in zip(want, got):
            assert np.array_equal(a, b)
        table, ring, words = got[0], got[1], got[5]
        cached = np.where(fresh < 0, 0, cached + fresh)
        held = [p for r in range(R) for p in table[r, :ref.up(int(cached[r]), page)]]
        free = [ring[(words[0] + i) % pages] for i in range(words[1])]
        assert sorted(held + free) == list(range(pages))
    dev.synchronize()


# ---- append ---------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("tokens,H,KV,hd,rot,src,dtype,page", [(1, 1, 1, 8, 8, "f32", "f32", 16), (5, 9, 3, 64, 64, "f32", "f32", 16), (7, 4, 2, 80, 80, "f32", "f16", 32), (3, 6, 2, 256, 256, "bf16", "bf16", 64),
                                                               (40, 32, 8, 128, 64, "f32", "bf16", 16), (11, 3, 3, 24, 8, "f16", "f32", 256), (6, 12, 12, 64, 0, "f16", "f16", 16), (300, 8, 1, 128, 128, "bf16", "f16", 128),
                                                               (9, 2, 1, 40, 40, "f16", "bf16", 16)])
def test_append(dev, tokens, H, KV, hd, rot, src, dtype, page):
    rng = np.random.default_rng(tokens * hd)
    pages, pad, most = ref.up(tokens, page) + 3, 4, 5000
    T = tokens + pad
    x, xn = put(dev, rng.normal(size=(T, (H + 2 * KV) * hd)), src)
    k, kn = put(dev, rng.normal(size=(pages, KV, page, hd)), dtype)
    v, vn = put(dev, rng.normal(size=(pages, KV, page, hd)), dtype)
    slots, positions = np.full(T, -1), np.full(T, -1)
    at = np.sort(rng.permutation(T)[:tokens])  # rows left out lie anywhere
    slots[at], positions[at] = rng.permutation(pages * page)[:tokens], rng.integers(0, most, tokens)
    positions[at[0]] = most - 1
    angle = np.arange(most)[:, None] * 10000.0 ** (-2.0 * np.arange(rot // 2) / max(rot, 1))
    cs = np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)
    rope = nn.Tensor.from_numpy(dev, cs) if rot else None
    out, on = put(dev, np.full((T, H, hd), 7.0), dtype)
    nn.paged_append(x, ints(dev, positions), ints(dev, slots), k, v, rope=rope, out=out)
    dev.synchronize()
    y = xn.astype(np.float64).reshape(T, H + 2 * KV, hd)
    size = np.abs(y)
    if rot:
        turn = cs[positions[at]].astype(np.float64)[:, None]
        y[at, :H + KV] = ref.rotate(y[at, :H + KV], turn)
        size[at, :H + KV] = ref.rotate(size[at, :H + KV], np.stack([np.abs(turn[..., 0]), -np.abs(turn[..., 1])], -1))
        h = rot // 2
        size[at, :H + KV, h:rot] = np.abs(size[at, :H + KV, h:rot])
        lo, hi = np.abs(xn.reshape(T, -1, hd)[at, :H + KV, :h]), np.abs(xn.reshape(T, -1, hd)[at, :H + KV, h:rot])
        size[at, :H + KV, h:rot] = hi * np.abs(turn[..., 0]) + lo * np.abs(turn[..., 1])
    # two products and a sum in f32, one rounding to the type (f16: to a multiple of 2^-24 below 2^-14)
    tol = 3 * 2.0 ** -24 * size + ref.EPS[dtype] * 1.001 * np.abs(y) + (2.0 ** -25 if dtype == "f16" else 0)
    wq, wk, wv = on.astype(np.float64), kn.astype(np.float64), vn.astype(np.float64)
    tq, tk, tv = np.zeros_like(wq), np.zeros_like(wk), np.zeros_like(wv)
    wq[at], tq[at] = y[at, :H], tol[at, :H]
    p, o = slots[at] // page, slots[at] % page
    wk[p, :, o], tk[p, :, o] = y[at, H:H + KV], tol[at, H:H + KV]
    wv[p, :, o], tv[p, :, o] = y[at, H + KV:], tol[at, H + KV:]
    for name, t, w, e in (("q", out, wq, tq), ("k", k, wk, tk), ("v", v, wv, tv)):
        bad = ~(np.abs(numbers(t) - w) <= e)
        assert not bad.any(), (name, np.argwhere(bad)[:3], np.abs(numbers(t) - w).max())


def test_append_in_place_without_queries_and_with_wide_rows(dev):
    """Through the C entry: queries turned in place in f32; no query output; parts of wider rows."""
    rng = np.random.default_rng(3)
    T, H, KV, hd, page, pages, ld = 6, 3, 2, 16, 16, 4, 3 * 16 + 2 * 2 * 16 + 20
    x0 = rng.normal(size=(T, ld)).astype(np.float32)
    cs = np.stack([np.cos(np.arange(50)[:, None] * np.ones(8)), np.sin(np.arange(50)[:, None] * np.ones(8))], -1).astype(np.float32)
    rope, slots, pos = nn.Tensor.from_numpy(dev, cs), ints(dev, rng.permutation(64)[:T]), ints(dev, np.arange(T) + 9)
    k_off, v_off = 3 * 16 + 2 * 16 + 12, 3 * 16 + 4  # values ahead of the keys
    got = []
    for q_out in (True, False):
        x = nn.Tensor.from_numpy(dev, x0)
        k, v = (nn.Tensor.from_numpy(dev, np.zeros((pages, KV, page, hd), np.float32)) for _ in range(2))
        dev.check(dev.L.ruai_paged_append(dev.ctx, nn.F32, x.ptr, ld, k_off, v_off, T, H, 16, rope.ptr, 50, pos.ptr, slots.ptr, nn.F32, k.ptr, v.ptr, pages, KV, page, hd,
                                          x.ptr if q_out else None, ld if q_out else 0))
        got.append((x.numpy(), k.numpy(), v.numpy()))
    (xa, ka, va), (xb, kb, vb) = got
    assert np.array_equal(xb, x0) and np.array_equal(ka, kb) and np.array_equal(va, vb) and np.array_equal(xa[:, 48:], x0[:, 48:])
    turn = cs[9:9 + T].astype(np.float64)[:, None]
    assert np.abs(xa[:, :48].reshape(T, H, hd) - ref.rotate(x0[:, :48].astype(np.float64).reshape(T, H, hd), turn)).max() < 1e-6
    s = slots.numpy()
    assert np.abs(ka[s // page, :, s % page] - ref.rotate(x0[:, k_off:k_off + 32].astype(np.float64).reshape(T, KV, hd), turn)).max() < 1e-6
    assert np.array_equal(va[s // page, :, s % page], x0[:, v_off:v_off + 32].reshape(T, KV, hd))


def test_append_out_of_range(dev):
    """A slot behind the pool, a position behind the rotations: left out and reported, the other rows are written."""
    x = nn.Tensor.from_numpy(dev, np.ones((4, 3 * 8), np.float32))
    rope = nn.Tensor.from_numpy(dev, np.stack([np.ones((5, 4)), np.zeros((5, 4))], -1).astype(np.float32))
    k, v = (nn.Tensor.from_numpy(dev, np.zeros((2, 1, 16, 8), np.float32)) for _ in range(2))
    out = nn.Tensor.from_numpy(dev, np.zeros((4, 1, 8), np.float32))
    nn.paged_append(x, ints(dev, [0, 5, -1, 4]), ints(dev, [32, 1, 2, 31]), k, v, rope=rope, out=out)
    with pytest.raises(nn.RuaiError, match="out of range"):
        dev.synchronize()
    assert out.numpy()[:, 0, 0].tolist() == [0, 0, 0, 1] and k.numpy().sum() == 8 and k.numpy()[1, 0, 15].all() and v.numpy().sum() == 8


# ---- attention ------------------------------------------------------------------------------------------------------------


def attend(dev, rng, cached, fresh, H, KV, hd, dtype, page, window=0, pad=3, scale=None, std=1.0, nan=True, most=None, mend=None):
    cached, fresh = np.asarray(cached), np.asarray(fresh)
    table, pages = lay_out(rng, cached + fresh, page)
    starts = np.concatenate([[0], np.cumsum(fresh)])
    T = int(starts[-1]) + pad
    kn, vn = rng.normal(size=(pages, KV, page, hd)) * std, rng.normal(size=(pages, KV, page, hd)) + 0.3
    if nan:  # what no request's positions cover may hold anything
        held = np.zeros((pages, page), bool)
        for r, n in enumerate(cached + fresh):
            for i in range(ref.up(int(n), page)):
                held[table[r, i], :min(page, int(n) - i * page)] = True
        junk = rng.choice([np.nan, np.inf, -np.inf], size=(pages, page))
        kn = np.where(held[:, None, :, None], kn, junk[:, None, :, None])
        vn = np.where(held[:, None, :, None], vn, junk[:, None, :, None])
    if mend is not None:
        mend(kn, vn, table)
    q, qn = put(dev, rng.normal(size=(T, H, hd)) * std, dtype)
    k, kn = put(dev, kn, dtype)
    v, vn = put(dev, vn, dtype)
    out, on = put(dev, np.full((T, H, hd), 7.0), dtype)
    most_fresh, most_len = most or (int(fresh.max()), int((cached + fresh).max()))
    scale = hd ** -0.5 if scale is None else scale
    nn.paged_attention(q, k, v, ints(dev, table), ints(dev, cached), ints(dev, starts), most_fresh, most_len, scale=scale, window=window, out=out)
    want, tol = ref.attention(qn, kn, vn, table, cached, starts, scale, window, dtype)
    return numbers(out), want, tol, on


def hold(got, want, tol, before, rows):
    assert np.array_equal(got[rows:], before[rows:]), "rows behind the last token"
    ok = (np.abs(got[:rows] - want[:rows]) <= tol[:rows]) | (np.isnan(want[:rows]) & np.isnan(got[:rows]))
    assert ok.all(), (np.argwhere(~ok)[:4].tolist(), (~ok).sum(), np.nanmax(np.abs(got[:rows] - want[:rows]) / np.maximum(tol[:rows], 1e-30)))


HEADS = [(1, 1, 8), (4, 2, 16), (9, 3, 64), (12, 12, 64), (8, 1, 128), (32, 8, 128), (5, 1, 80), (16, 4, 80), (6, 2, 256), (14, 2, 40), (3, 1, 136)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,KV,hd", HEADS)
def test_attention_single_tokens(dev, H, KV, hd, dtype):
    rng = np.random.default_rng(hd + H)
    cached = [0, 1, 15, 16, 17, 63, 64, 130, 255, 300, 31, 47]
    r = attend(dev, rng, cached, [1] * len(cached), H, KV, hd, dtype, 16)
    dev.synchronize()
    hold(*r, len(cached))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,KV,hd", HEADS)
def test_attention_few_tokens(dev, H, KV, hd, dtype):
    rng = np.random.default_rng(hd + H + 1)
    cached, fresh = [0, 10, 200, 15, 16, 77, 5], [5, 1, 4, 2, 0, 9, 3]
    r = attend(dev, rng, cached, fresh, H, KV, hd, dtype, 32)
    dev.synchronize()
    hold(*r, sum(fresh))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,KV,hd,window", [(4, 2, 16, 0), (9, 3, 64, 0), (8, 8, 64, 50), (8, 1, 128, 0), (16, 4, 128, 200), (5, 1, 80, 0), (6, 2, 256, 33), (14, 2, 40, 0), (3, 1, 136, 0), (2, 1, 96, 1)])
def test_attention_chunks(dev, H, KV, hd, window, dtype):
    """Chunks beside single tokens, at lengths around every tile's edge."""
    rng = np.random.default_rng(hd + H + 2)
    cached, fresh = [0, 100, 0, 333, 128, 1, 64], [130, 1, 64, 65, 127, 0, 200]
    r = attend(dev, rng, cached, fresh, H, KV, hd, dtype, 16, window=window)
    dev.synchronize()
    hold(*r, sum(fresh))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("fresh", [1, 3, 70])
def test_attention_page_sizes(dev, page, fresh, dtype):
    rng = np.random.default_rng(page + fresh)
    cached = [0, page - 1, page, 3 * page + 5, 2 * page - fresh % page]
    r = attend(dev, rng, cached, [fresh] * 5, 8, 2, 64, dtype, page)
    dev.synchronize()
    hold(*r, 5 * fresh)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("window", [1, 2, 16, 17, 63, 64, 65, 300, 5000])
@pytest.mark.parametrize("fresh", [1, 6, 150])
def test_attention_windows(dev, window, fresh, dtype):
    rng = np.random.default_rng(window + fresh)
    cached = [0, 40, 64, 500]
    r = attend(dev, rng, cached, [fresh] * 4, 8, 2, 64, dtype, 16, window=window)
    dev.synchronize()
    hold(*r, 4 * fresh)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cached,fresh,H,KV,hd,window", [(20000, 1, 8, 2, 128, 0), (9000, 4, 4, 1, 64, 0), (5000, 1, 32, 8, 128, 700), (3000, 40, 8, 2, 64, 0), (4000, 130, 4, 1, 128, 0), (6000, 2, 6, 2, 256, 0)])
def test_attention_long_caches(dev, cached, fresh, H, KV, hd, window, dtype):
    """Few rows over many keys: the keys of a request are shared out and joined."""
    rng = np.random.default_rng(cached)
    r = attend(dev, rng, [cached, 5, cached // 3], [fresh, 1, fresh], H, KV, hd, dtype, 16, window=window)
    dev.synchronize()
    hold(*r, 2 * fresh + 1)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("fresh", [1, 5, 100])
def test_attention_large_scores(dev, fresh, dtype):
    """Scores of tens: a row is nearly one key; and rising ones, which move the maximum at every tile."""
    rng = np.random.default_rng(fresh)

    def rising(k, v, table):
        for i, pg in enumerate(table[1][table[1] >= 0]):
            k[pg] *= 1 + 0.5 * i

    for mend in (None, rising):
        r = attend(dev, rng, [300, 700], [fresh] * 2, 8, 2, 64, dtype, 16, std=2.5, mend=mend)
        dev.synchronize()
        hold(*r, 2 * fresh)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("fresh", [1, 6, 90])
@pytest.mark.parametrize("what", ["inf value", "nan value", "nan key", "-inf key", "inf key"])
def test_attention_infinities_and_nan(dev, fresh, what, dtype):
    """In a key that some rows see and others do not: the others' results are as if it were not there."""
    rng = np.random.default_rng(fresh)
    cached = 100
    at = cached + (fresh - 1) // 2  # seen by the second half of the rows

    def mend(k, v, table):
        pg, o = table[0, at // 16], at % 16
        if what.endswith("value"):
            v[pg, :, o, 3] = float(what.split()[0])
        else:
            k[pg, :, o, :] = 0.0
            k[pg, 1, o, 2] = float(what.split()[0])

    got, want, tol, before = attend(dev, rng, [cached, 10], [fresh, 1], 8, 2, 64, dtype, 16, mend=mend, pad=0)
    dev.synchronize()
    with np.errstate(invalid="ignore"):
        ok = (np.abs(got - want) <= tol) | (np.isnan(want) & np.isnan(got)) | (got == want)
    if what == "inf key":  # scores of +inf: NaN, whatever the maximum of the others
        ok |= ~np.isfinite(want) & ~np.isfinite(got)
    assert ok.all(), (np.argwhere(~ok)[:4].tolist(), (~ok).sum())


def test_attention_scale_zero_negative_and_far_queries(dev):
    rng = np.random.default_rng(9)
    for scale in (0.0, -0.3, 3.0):
        for dtype in ("f32", "bf16"):
            for fresh in (1, 70):
                r = attend(dev, rng, [130, 20], [fresh, fresh], 4, 2, 32, dtype, 16, scale=scale)
                dev.synchronize()
                hold(*r, 2 * fresh)


def test_attention_many_requests(dev):
    rng = np.random.default_rng(10)
    R = 1500
    cached, fresh = rng.integers(0, 60, R), (rng.random(R) < 0.7).astype(int)
    fresh[700] = 90
    r = attend(dev, rng, cached, fresh, 4, 2, 32, "bf16", 16)
    dev.synchronize()
    hold(*r, int(fresh.sum()))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fresh", [1, 80])
def test_attention_leaves_out_what_is_out_of_range(dev, fresh, dtype):
    """Lengths beyond the bounds or the table, starts that run backwards, pages outside the pool: reported; other requests are served."""
    rng = np.random.default_rng(11)
    q, qn = put(dev, rng.normal(size=(4 * fresh, 2, 16)), dtype)
    k, kn = put(dev, rng.normal(size=(12, 1, 16, 16)), dtype)
    v, vn = put(dev, rng.normal(size=(12, 1, 16, 16)), dtype)
    width = ref.up(20 + fresh, 16)
    table = np.tile(np.arange(width), (4, 1))
    starts = np.arange(5) * fresh
    for change in ("cached", "long", "table", "page", "negative page"):
        cached, tab = np.full(4, 20), table.copy()
        if change == "cached":
            cached[2] = -5
        if change == "long":
            cached[2] = 25  # beyond most_len, and with it beyond the table
        if change == "table":
            cached[2] = 16 * width
        if "page" in change:
            tab[2, 0] = -1 if change == "negative page" else 12
        out, before = put(dev, np.full((4 * fresh, 2, 16), 7.0), dtype)
        nn.paged_attention(q, k, v, ints(dev, tab), ints(dev, cached), ints(dev, starts), fresh, 10**6 if change == "table" else 20 + fresh, out=out)
        with pytest.raises(nn.RuaiError, match="out of range"):
            dev.synchronize()
        want, tol = ref.attention(qn, kn, vn, table, np.full(4, 20), starts, 0.25, 0, dtype)
        got = numbers(out)
        for r in (0, 1, 3):
            rows = slice(r * fresh, (r + 1) * fresh)
            assert (np.abs(got[rows] - want[rows]) <= tol[rows]).all(), change
        if "page" not in change:
            assert np.array_equal(got[2 * fresh:3 * fresh], before[2 * fresh:3 * fresh]), change


def test_entry_points_check_their_arguments(dev):
    t = nn.Tensor.from_numpy(dev, np.zeros(4096, np.float32))
    L, p, odd = dev.L, t.ptr, C.c_void_p(t.ptr.value + 4)
    plan = dict(cached=p, fresh=p, R=1, tokens=1, page=16, table=p, ld=1, ring=p, pages=4, win=p, wout=p, starts=p, pos=p, slots=p)
    append = dict(xd=0, x=p, ld=48, k=16, v=32, tokens=1, H=1, rot=16, rope=p, most=4, pos=p, slots=p, d=0, kp=p, vp=p, pages=1, KV=1, page=16, hd=16, q=p, q_ld=16)
    attn = dict(d=0, q=p, q_ld=16, kp=p, vp=p, pages=1, KV=1, page=16, hd=16, table=p, ld=1, cached=p, starts=p, R=1, tokens=1, H=1, scale=1.0, window=0, fresh=1, len=1, out=p, out_ld=16)
    for fn, base, changes in ((L.ruai_page_plan, plan, [dict(page=24), dict(page=8), dict(page=512), dict(R=0), dict(R=8193), dict(tokens=262145), dict(ld=0), dict(pages=0), dict(pages=1 << 28), dict(slots=None), dict(win=None), dict(wout=odd)]),
                              (L.ruai_paged_append, append, [dict(xd=3), dict(d=-1), dict(page=20), dict(hd=12), dict(hd=264), dict(hd=0), dict(KV=0), dict(pages=0), dict(pages=1 << 28), dict(rot=0), dict(rot=12),
                                                            dict(rot=24), dict(most=0), dict(ld=46), dict(ld=40), dict(k=18), dict(q_ld=12), dict(x=odd), dict(q=odd), dict(kp=odd), dict(rope=odd), dict(slots=None),
                                                            dict(pos=None)]),
                              (L.ruai_paged_attention, attn, [dict(d=5), dict(page=17), dict(hd=20), dict(KV=0), dict(H=0), dict(H=3, KV=2), dict(H=257, q_ld=8192, out_ld=8192), dict(q_ld=18), dict(q_ld=12), dict(out_ld=8),
                                                              dict(q=odd), dict(out=odd), dict(vp=odd), dict(ld=0), dict(R=8193), dict(tokens=262145), dict(len=1 << 30), dict(scale=float("nan")), dict(table=None),
                                                              dict(out=None)])):
        for change in changes:
            rc = fn(dev.ctx, *{**base, **change}.values())
            assert rc in (1, 6), (fn.__name__, change, rc)
    # nothing to do is no error
    assert L.ruai_paged_append(dev.ctx, *{**append, "tokens": 0}.values()) == 0
    assert L.ruai_paged_attention(dev.ctx, *{**attn, "tokens": 0}.values()) == 0 and L.ruai_paged_attention(dev.ctx, *{**attn, "R": 0}.values()) == 0
    dev.synchronize()


# ---- together -------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_steps_of_a_serving_loop(dev, dtype):
    """Plan, append, attention over several steps with requests that come, grow and end, against all of it in float64."""
    rng = np.random.default_rng(12)
    R, H, KV, hd, page, pages, width = 5, 6, 2, 64, 16, 64, 20
    cs = np.stack([np.cos(np.arange(400)[:, None] * 0.1 ** np.arange(32)), np.sin(np.arange(400)[:, None] * 0.1 ** np.arange(32))], -1).astype(np.float32)
    rope = nn.Tensor.from_numpy(dev, cs)
    k, kn = put(dev, np.full((pages, KV, page, hd), np.nan), dtype)
    v, vn = put(dev, np.full((pages, KV, page, hd), np.nan), dtype)
    kn, vn = kn.astype(np.float64), vn.astype(np.float64)
    table, ring, words = ints(dev, np.full((R, width), -1)), ints(dev, rng.permutation(pages)), ints(dev, [0, pages, 0])
    cached = np.zeros(R, np.int64)
    for step, fresh in enumerate(([90, 0, 3, 0, 17], [1, 33, 1, 0, 1], [1, 1, 1, 70, 1], [-1, 1, 5, 1, 1], [100, 1, 1, -1, 1], [1, 1, 0, 2, 1])):
        fresh = np.array(fresh)
        T = int(fresh.clip(0).sum()) + 2
        dc, df = ints(dev, cached), ints(dev, fresh)
        plan = nn.page_plan(dc, df, table, ring, words, page, tokens=T)
        x, xn = put(dev, rng.normal(size=(T, (H + 2 * KV) * hd)), dtype)
        out, before = put(dev, np.full((T, H, hd), 7.0), dtype)
        q = nn.paged_append(x, plan.positions, plan.slots, k, v, rope=rope)
        nn.paged_attention(q, k, v, table, dc, plan.starts, int(fresh.max()), int((cached + fresh.clip(0)).max()), out=out)
        words = plan.words
        dev.synchronize()
        # what the GPU wrote into the pages is what the attention below is held to; append has its own test
        want, tol = ref.attention(numbers(q), numbers(k), numbers(v), table.numpy(), np.where(fresh < 0, 0, cached), plan.starts.numpy(), hd ** -0.5, 0, dtype)
        hold(numbers(out), want, tol, before, T - 2)
        cached = np.where(fresh < 0, 0, cached + fresh)
    assert words.numpy()[1] == pages - sum(ref.up(int(n), page) for n in cached)


def test_calls_repeat_their_bits(dev):
    """The same call twice, and beside calls of other shapes in between: no result depends on what a workspace held."""
    rng = np.random.default_rng(13)
    shapes = [([3000], [1], 8, 2, 128, "bf16"), ([700, 30], [50, 1], 8, 2, 64, "f16"), ([900], [200], 4, 1, 128, "bf16"), ([2000, 2], [3, 1], 8, 2, 64, "f32"), ([10], [150], 8, 2, 64, "f32")]
    first = [attend(dev, np.random.default_rng(i), *s[:5], s[5], 16)[0] for i, s in enumerate(shapes)]
    for i in rng.permutation(len(shapes) * 3) % len(shapes):
        s = shapes[i]
        again = attend(dev, np.random.default_rng(i), *s[:5], s[5], 16)[0]
        assert np.array_equal(first[i], again), i


# ---- what calls may be ------------------------------------------------------------------------------------------------------


def test_plan_refuses_more_pages_back_than_there_is_room_for(dev):
    """Free pages and those that come back are more than the ring holds: refused, whatever is given out in the same step."""
    table, ring = np.array([[0, 1, 2, 3], [4, 5, -1, -1]]), np.arange(10)
    got = run_plan(dev, [64, 16], [-1, 17], table, ring, [0, 7, 0], 16, 20)
    with pytest.raises(nn.RuaiError, match="page plan was refused"):
        dev.synchronize()
    assert np.array_equal(got[0], table) and np.array_equal(got[1], ring) and got[5].tolist() == [0, 7, 0]


def test_entry_points_refuse_overlaps_and_widths(dev):
    t = nn.Tensor.from_numpy(dev, np.zeros(4096, np.float32))
    L, p = dev.L, t.ptr
    append = dict(xd=nn.F32, x=p, ld=48, k=16, v=32, tokens=1, H=1, rot=16, rope=None, most=0, pos=None, slots=p, d=nn.F32, kp=p, vp=p, pages=1, KV=1, page=16, hd=16, q=None, q_ld=0)
    for change in (dict(q=p, q_ld=16), dict(q=p, q_ld=48, d=nn.F16), dict(H=2**32 - 1), dict(H=2**28)):
        assert L.ruai_paged_append(dev.ctx, *{**append, **change}.values()) in (1, 6), change
    with pytest.raises(nn.RuaiError, match="apart"):
        q, pages = (nn.Tensor.from_numpy(dev, np.zeros(n, np.float32)) for n in ((1, 1, 16), (1, 1, 16, 16)))
        nn.paged_attention(q, pages, pages, ints(dev, [[0]]), ints(dev, [0]), ints(dev, [0, 1]), 1, 1, out=q)
    dev.synchronize()


@pytest.fixture()
def capturing(dev):
    from test_gpu_ops import Capturing
    c = Capturing()
    yield c
    c.close()


@pytest.mark.parametrize("warm", [False, True])
@pytest.mark.parametrize("cached,fresh,H,KV,hd,dtype", [(3000, 1, 8, 2, 128, "bf16"), (900, 200, 4, 1, 128, "bf16"), (2000, 3, 8, 2, 64, "f32"), (10, 400, 8, 2, 64, "f32")])
def test_attention_in_a_graph_whose_scratch_has_moved(capturing, cached, fresh, H, KV, hd, dtype, warm):
    """Captured on a fresh context and on one whose scratch has grown for the kernel; replayed with other queries after the scratch has moved."""
    d, rng = capturing.dev, np.random.default_rng(17)
    width = ref.up(cached + fresh, 16)
    (k, kn), (v, vn) = (put(d, rng.normal(size=(width + 1, KV, 16, hd)), dtype) for _ in range(2))
    (q, qn), on = put(d, rng.normal(size=(fresh, H, hd)), dtype), ref.stored(rng.normal(size=(fresh, H, hd)), dtype)[1]
    table, lens, starts = rng.permutation(width + 1)[None, :width], np.array([cached]), np.array([0, fresh])
    args = (k, v, ints(d, table), ints(d, lens), ints(d, starts), fresh, cached + fresh)
    out, before = put(d, np.full((fresh, H, hd), 7.0), dtype)
    if warm:
        nn.paged_attention(q, *args, out=out)
        d.synchronize()
    capturing.begin()
    try:
        nn.paged_attention(q, *args, out=out)
    finally:
        assert capturing.end() == 0

    def replayed(queries):
        capturing.replay()
        want, tol = ref.attention(queries, kn, vn, table, lens, starts, hd ** -0.5, 0, dtype)
        hold(numbers(out), want, tol, before, fresh)

    replayed(qn)
    # a prompt in f32 whose pieces take more scratch than any call before
    far, pages = nn.Tensor.from_numpy(d, np.zeros((4000, 8, 128), np.float32)), nn.Tensor.from_numpy(d, np.zeros((500, 8, 16, 128), np.float32))
    nn.paged_attention(far, pages, pages, ints(d, np.arange(500)[None]), ints(d, [4000]), ints(d, [0, 4000]), 4000, 8000)
    d.synchronize()
    changed = ref.stored(on, dtype)[0]
    d.check(d.L.ruai_memcpy_h2d(d.ctx, q.ptr, changed.ctypes.data_as(C.c_void_p), q.nbytes))
    replayed(on)
    for t in (k, v, q, out, far, pages, *args[2:5]):
        t.free()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,KV,hd", [(4, 2, 72), (6, 1, 104), (8, 8, 120), (5, 1, 88), (24, 1, 64), (48, 1, 72), (64, 1, 128), (100, 1, 64), (128, 1, 64), (129, 1, 64), (256, 1, 16)])
def test_attention_odd_heads_and_many_per_key(dev, H, KV, hd, dtype):
    """Heads that are no multiple of 16, and as many query heads per key as rows of a tile, fewer and more."""
    rng = np.random.default_rng(21)
    for cached, fresh, window in (([130, 0, 33], [1, 1, 1], 0), ([0, 200, 17, 5], [70, 3, 131, 0], 0), ([300], [129], 50)):
        got, want, tol, before = attend(dev, rng, cached, fresh, H, KV, hd, dtype, 16, window=window)
        hold(got, want, tol, before, sum(fresh))
    dev.synchronize()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,KV,hd,cached,fresh", [(8, 2, 64, [700, 3], [1, 1]), (8, 2, 128, [0, 100], [300, 1]), (5, 1, 72, [50], [90])])
def test_attention_rows_wider_than_the_heads(dev, H, KV, hd, cached, fresh, dtype):
    """q and out as columns of wider tensors: what lies between the rows is neither read into results nor written."""
    rng = np.random.default_rng(23)
    cached, fresh = np.array(cached), np.array(fresh)
    table, pages = lay_out(rng, cached + fresh, 16)
    starts = np.concatenate([[0], np.cumsum(fresh)])
    T, wide = int(starts[-1]), H * hd
    x = np.full((T, wide + 24), np.nan)
    x[:, 8:8 + wide] = rng.normal(size=(T, wide))
    q, qn = put(dev, x, dtype)
    (k, kn), (v, vn) = (put(dev, rng.normal(size=(pages, KV, 16, hd)), dtype) for _ in range(2))
    out, _ = put(dev, np.full((T + 1, wide + 40), 7.0), dtype)
    size, t, c, s = q.np_dtype.itemsize, ints(dev, table), ints(dev, cached), ints(dev, starts)
    dev.check(dev.L.ruai_paged_attention(dev.ctx, RD[dtype], C.c_void_p(q.ptr.value + 8 * size), wide + 24, k.ptr, v.ptr, pages, KV, 16, hd, t.ptr, table.shape[1], c.ptr, s.ptr, len(cached), T, H,
                                         hd ** -0.5, 0, int(fresh.max()), int((cached + fresh).max()), C.c_void_p(out.ptr.value + 16 * size), wide + 40))
    dev.synchronize()
    got = numbers(out)
    want, tol = ref.attention(qn[:, 8:8 + wide].reshape(T, H, hd), kn, vn, table, cached, starts, hd ** -0.5, 0, dtype)
    hold(got[:T, 16:16 + wide].reshape(T, H, hd), want, tol, want[:T], T)
    got[:T, 16:16 + wide] = 7
    assert (got == 7).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_two_graphs_of_one_context_in_turn(capturing, dtype):
    """Two captured calls of other shapes share a workspace; replayed in turn, each gives the bits of its call by itself."""
    d, rng = capturing.dev, np.random.default_rng(29)
    calls, want, keep = [], [], []
    for cached, fresh, H, KV, hd in ((4000, 1, 8, 2, 128), (700, 150, 8, 2, 64)):
        width = ref.up(cached + fresh, 16)
        k, v = (put(d, rng.normal(size=(width, KV, 16, hd)), dtype)[0] for _ in range(2))
        q, out = (put(d, rng.normal(size=(fresh, H, hd)), dtype)[0] for _ in range(2))
        args = (q, k, v, ints(d, rng.permutation(width)[None]), ints(d, [cached]), ints(d, [0, fresh]), fresh, cached + fresh)
        nn.paged_attention(*args, out=out)
        want.append(out.numpy())
        calls.append((args, out))
        keep += [k, v, q, out, *args[3:6]]
    graphs = []
    for args, out in calls:
        capturing.begin()
        try:
            nn.paged_attention(*args, out=out)
        finally:
            assert capturing.end() == 0
        capturing.replay()
        graphs.append((capturing.graph, capturing.exec))
        capturing.graph, capturing.exec = C.c_void_p(), C.c_void_p()
    for turn in range(6):
        which = (0, 1, 1, 0, 1, 0)[turn]
        out = calls[which][1]
        d.check(d.L.ruai_memcpy_h2d(d.ctx, out.ptr, np.zeros_like(want[which]).ctypes.data_as(C.c_void_p), out.nbytes))
        assert capturing.cu.cuGraphLaunch(graphs[which][1], capturing.stream) == 0
        d.synchronize()
        assert np.array_equal(out.numpy(), want[which]), turn
    for graph, ex in graphs:
        capturing.cu.cuGraphExecDestroy(ex)
        capturing.cu.cuGraphDestroy(graph)
    for t in keep:
        t.free()


def attend_to(dev, q, k, v, table, cached, fresh, dtype, scale, window=0):
    """One call on these numbers: (what it wrote, what the inputs hold)."""
    starts = np.concatenate([[0], np.cumsum(fresh)])
    (q, qn), (k, kn), (v, vn) = (put(dev, x, dtype) for x in (q, k, v))
    out, _ = put(dev, np.full(qn.shape, 7.0), dtype)
    nn.paged_attention(q, k, v, ints(dev, table), ints(dev, cached), ints(dev, starts), int(np.max(fresh)), int(np.max(np.add(cached, fresh))), scale=scale, window=window, out=out)
    return numbers(out), (qn, kn, vn, table, cached, starts, scale, window, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("fresh", [1, 40])
@pytest.mark.parametrize("what", ["nan query", "inf query", "nan keys", "-inf keys", "inf values", "nan first key"])
def test_attention_infinities_and_nan_in_parts_of_long_requests(dev, what, fresh, dtype):
    """A request so long that its keys are shared out: parts without a finite score are not lost where the parts are joined."""
    rng = np.random.default_rng(fresh)
    H, KV, hd, cached, page = 8, 2, 64, 2500, 16
    n = ref.up(cached + fresh, page)
    q, k, v = (rng.normal(size=s) for s in ((fresh, H, hd), (n, KV, page, hd), (n, KV, page, hd)))
    table = rng.permutation(n)[None]
    if what == "nan query":
        q[fresh // 2, 3] = np.nan
    if what == "inf query":
        q[fresh // 2, 3, 5] = np.inf
    if what == "nan keys":
        k[table[0, 96:]] = np.nan  # positions 1536 and up
    if what == "nan first key":
        k[table[0, 0], 1, 0, 7] = np.nan
    if what == "-inf keys":  # weigh nothing, whatever their values are
        q[..., 0], k[table[0, 96:, None], 0, :, 0] = np.abs(q[..., 0]) + 0.1, -np.inf
        v[table[0, 130], 0] = np.inf
    if what == "inf values":
        v[table[0, 100], 1, 3, 9], v[table[0, 20], 0, 3, 9] = np.inf, -np.inf
    got, args = attend_to(dev, q, k, v, table, np.array([cached]), np.array([fresh]), dtype, hd ** -0.5)
    dev.synchronize()
    want, tol = ref.attention(*args)
    with np.errstate(invalid="ignore"):
        ok = (np.abs(got - want) <= tol) | (np.isnan(want) & np.isnan(got)) | (got == want)
    assert ok.all(), (np.argwhere(~ok)[:4].tolist(), (~ok).sum())
    assert np.isnan(want).any() or "nan" not in what


@pytest.mark.parametrize("R,fresh", [(80, 1), (40, 26)])
@pytest.mark.parametrize("bits", [16, 20, 24])
@pytest.mark.parametrize("spread", [0.0, 0.3])
def test_attention_tail_behind_a_key_with_nearly_all_weight(dev, spread, bits, R, fresh):
    """f16, one key `bits` powers of two above 600 others and without a value: the others are the result, and keep their bits.
    More requests than the GPU runs at a time, so that the keys of most are not shared out.

    Weights reach the values as f16, the largest as 2^7 at least, so that one is off by half a step, 2^-11 of itself, or by 2^-25 where it is
    below 2^-14: 2^-32 of the largest.  The scores themselves are off as everywhere (paged_cases.attention)."""
    rng = np.random.default_rng(bits)
    KV, hd, cached, page = 4, 64, 600, 16
    n = ref.up(cached + fresh, page)
    q, k, v = np.zeros((R * fresh, KV, hd)), np.zeros((R * n, KV, page, hd)), 100 + 20 * rng.normal(size=(R * n, KV, page, hd))
    q[..., 0], q[..., 1] = 1, 1
    k[..., 1] = spread * rng.normal(size=(R * n, KV, page))
    table = rng.permutation(R * n).reshape(R, n)
    k[table[:, 3], :, 5, 0], k[table[:, 3], :, 5, 1], v[table[:, 3], :, 5] = bits * np.log(2), 0, 0
    got, args = attend_to(dev, q, k, v, table, np.full(R, cached), np.full(R, fresh), "f16", 1.0)
    dev.synchronize()
    want, f32_tol = ref.attention(*args[:-1], "f32")
    size = np.abs(want)  # the values are positive
    tail = np.abs(args[2].astype(np.float64))[table].sum((1, 3)).repeat(fresh, 0) * 2.0 ** -32  # the weights' sum is the largest at least
    tol = f32_tol + size * 2.0 ** -11 + size * 2.0 ** -11 * 1.01 + tail + 2.0 ** -25
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / size).max()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_graphs_captured_between_growths_of_the_scratch(capturing, dtype):
    """Calls captured one after the other while the scratch grows in between, some of its blocks captured and some not: each replays its bits."""
    d, rng = capturing.dev, np.random.default_rng(31)
    cached, fresh, H, KV, hd = 3000, 1, 8, 2, 64
    width = ref.up(cached + fresh, 16)
    k, v = (put(d, rng.normal(size=(width, KV, 16, hd)), dtype)[0] for _ in range(2))
    q, out = (put(d, rng.normal(size=(fresh, H, hd)), dtype)[0] for _ in range(2))
    args = (q, k, v, ints(d, rng.permutation(width)[None]), ints(d, [cached]), ints(d, [0, fresh]), fresh, cached + fresh)
    nn.paged_attention(*args, out=out)
    want, graphs, keep = out.numpy(), [], [k, v, q, out, *args[3:6]]
    for i, rows in enumerate((700, 1100, 1700, 2600, 4000)):
        far, pages = nn.Tensor.from_numpy(d, np.zeros((rows, 8, 128), np.float32)), nn.Tensor.from_numpy(d, np.zeros((ref.up(rows, 16), 8, 16, 128), np.float32))
        nn.paged_attention(far, pages, pages, ints(d, np.arange(ref.up(rows, 16))[None]), ints(d, [0]), ints(d, [0, rows]), rows, rows)
        d.synchronize()
        keep += [far, pages]
        if i % 2 == 0:
            capturing.begin()
            try:
                nn.paged_attention(*args, out=out)
            finally:
                assert capturing.end() == 0
            capturing.replay()
            graphs.append((capturing.graph, capturing.exec))
            capturing.graph, capturing.exec = C.c_void_p(), C.c_void_p()
        for _, ex in graphs:
            d.check(d.L.ruai_memcpy_h2d(d.ctx, out.ptr, np.zeros_like(want).ctypes.data_as(C.c_void_p), out.nbytes))
            assert capturing.cu.cuGraphLaunch(ex, capturing.stream) == 0
            d.synchronize()
            assert np.array_equal(out.numpy(), want), i
    for graph, ex in graphs:
        capturing.cu.cuGraphExecDestroy(ex)
        capturing.cu.cuGraphDestroy(graph)
    for t in keep:
        t.free()


@pytest.mark.parametrize("most_len", [4000, 33000])
def test_attention_f32_chunks_whose_bound_fills_the_scratch(dev, most_len):
    """Chunks in f32 with room for so many positions that the pieces of seven requests of the twelve are made at a time, or those of none."""
    rng = np.random.default_rng(37)
    cached, fresh = np.full(12, 30), np.ones(12, int)
    cached[[1, 10]], fresh[[1, 10]] = (500, 61), (130, 129)
    got, want, tol, before = attend(dev, rng, cached, fresh, 8, 8, 128, "f32", 16, most=(130, most_len))
    dev.synchronize()
    hold(got, want, tol, before, int(fresh.sum()))
