"""The paged cache's operators in float64 numpy, with how far a result in a given type may be off."""
import numpy as np

EPS = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step, relative


def up(a, b):
    return -(-a // b)


def to_bf16(a):
    b = np.ascontiguousarray(a, np.float32).view(np.uint32)
    nan = np.isnan(a)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(nan, np.uint16(0x7FC0), r)


def from_bf16(r):
    return (np.asarray(r, np.uint16).astype(np.uint32) << 16).view(np.float32)


def stored(a, dtype):
    """What a tensor of the type holds, as the library takes it and as numbers."""
    with np.errstate(over="ignore"):
        if dtype == "f32":
            s = np.asarray(a, np.float32)
            return s, s
        if dtype == "f16":
            s = np.asarray(a, np.float32).astype(np.float16)
            return s, s.astype(np.float32)
    s = to_bf16(np.asarray(a, np.float32))
    return s, from_bf16(s)


def plan(cached, fresh, table, ring, words, page, tokens):
    """(table, ring, starts, positions, slots, words) after a plan, or None where it is refused."""
    table, ring, pages = table.copy(), ring.copy(), len(ring)
    first, free = int(words[0]), int(words[1])
    starts, positions, slots = [0], np.full(tokens, -1), np.full(tokens, -1)
    taken, back = 0, []
    for r, (c, f) in enumerate(zip(cached, fresh)):
        held = up(int(c), page)
        if up(int(c) + max(int(f), 0), page) > table.shape[1]:
            return None
        if f < 0:
            back += table[r, :held].tolist()
        for i in range(held, up(int(c) + max(int(f), 0), page)):
            if taken < free:
                table[r, i] = ring[(first + taken) % pages]
            taken += 1
        starts.append(starts[-1] + max(int(f), 0))
        if starts[-1] > tokens:
            return None
    if taken > free:
        return None
    for k, p in enumerate(back):
        ring[(first + free + k) % pages] = p
    for r, (c, f) in enumerate(zip(cached, fresh)):
        for i in range(max(int(f), 0)):
            p = int(c) + i
            positions[starts[r] + i] = p
            slots[starts[r] + i] = table[r, p // page] * page + p % page
    return table, ring, np.array(starts), positions, slots, np.array([(first + taken) % pages, free - taken + len(back), 0])


def rotate(x, cs):
    """x [.., hd] turned by cs [.., rot / 2, 2], which broadcast."""
    h = cs.shape[-2]
    a, b, c, s = x[..., :h], x[..., h:2 * h], cs[..., 0], cs[..., 1]
    return np.concatenate([a * c - b * s, b * c + a * s, x[..., 2 * h:]], -1)


def attention(q, k, v, table, cached, starts, scale, window, dtype):
    """out [tokens, H, hd] in float64 (NaN for rows of no request) and its tolerance.

    A score is a sum of hd products, each rounded in 2^-23 at most (f32, or pieces of 22 bits and a sum that truncates), a row's sums
    have as many terms as it sees keys, and in 16 bits the weights are rounded once before they meet the values; f16 weights below
    2^-14 of the largest by 2^-25 of it.  A score off by d scales its weight by e^d, in the numerator and in the sum."""
    pages, KV, page, hd = k.shape
    T, H, _ = q.shape
    rep = H // KV
    out, tol = np.full((T, H, hd), np.nan), np.zeros((T, H, hd))
    with np.errstate(invalid="ignore"):  # NaN where nothing is held
        k, v, q = (np.asarray(x, np.float64) for x in (k, v, q))
    for r in range(len(cached)):
        c, t0, t1 = int(cached[r]), int(starts[r]), int(starts[r + 1])
        if t0 == t1:
            continue
        n = c + t1 - t0
        pg = table[r, :up(n, page)]
        K = k[pg].transpose(1, 0, 2, 3).reshape(KV, -1, hd)[:, :n]
        V = v[pg].transpose(1, 0, 2, 3).reshape(KV, -1, hd)[:, :n]
        for t in range(t0, t1):
            p = c + t - t0
            lo = max(0, p + 1 - window) if window else 0
            with np.errstate(all="ignore"):
                kk, vv = K[:, lo:p + 1].repeat(rep, 0), V[:, lo:p + 1].repeat(rep, 0)
                s = np.einsum("hd,hkd->hk", q[t], kk) * scale
                d = np.einsum("hd,hkd->hk", np.abs(q[t]), np.abs(kk)).max(-1, initial=0) * abs(scale) * (hd + 8) * 2.0 ** -23
                m = s.max(-1, keepdims=True)
                w = np.exp(s - np.where(np.isfinite(m), m, 0))
                l = w.sum(-1, keepdims=True)
                w = w / l
                vv = np.where((w == 0)[..., None], 0, vv)  # a key that weighs nothing, whatever its value
                out[t] = np.einsum("hk,hkd->hd", w, vv)
                size = np.einsum("hk,hkd->hd", w, np.abs(vv))
                tol[t] = size * (2 * d + (s.shape[-1] + 32) * 2.0 ** -24)[:, None]
                if dtype != "f32":
                    tol[t] += size * EPS[dtype] + np.abs(out[t]) * EPS[dtype] * 1.01
                if dtype == "f16":
                    tol[t] += 2.0 ** -25 * np.abs(vv).sum(1) / l + 2.0 ** -25
    return out, tol
