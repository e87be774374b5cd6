"""The paged cache of a serving batch as timed cases: block tables and slot maps from request lengths (`plan`), rotation and the
writing of keys and values (`append`), and attention of every request's new tokens over its pages (`attention`).

Requests have lengths of their own, drawn from the case alone; values and the order of the pages in the pool come from the
seed.  With `own` the calls go through `ruai_b200.nn`, otherwise the operators are computed by elementary torch operations.
"""
import math

import numpy as np
import torch

from ruai_b200 import nn

own = False

_NP = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}
_TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_DTYPE = {"f32": nn.F32, "f16": nn.F16, "bf16": nn.BF16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
# query heads, key heads, head width: the 8B, 1.1B and 135M Llama shapes, GPT-2, one key head for all, odd widths
HEADS = [(32, 8, 128), (32, 4, 64), (9, 3, 64), (12, 12, 64), (8, 1, 128), (16, 4, 80), (6, 2, 256)]


def listed():
    return [
        # an ordinary decoding step of a small server: 64 requests, a token each, some begin a page
        dict(name="plan-64-steps", kind="plan", R=64, fresh=1, prompts=0, ended=2, most=4096, page=16, pad=0, salt=1),
        # a large scheduler step: two thousand requests, most decode, some bring prompts, some have ended
        dict(name="plan-2000-mixed", kind="plan", R=2000, fresh=1500, prompts=40, ended=90, most=8000, page=32, pad=500, salt=2),
        # the smallest write: one token of the smallest Llama, kept in f32
        dict(name="append-1-f32", kind="append", tokens=1, pad=0, H=9, KV=3, hd=64, rot=64, src="f32", dtype="f32", page=16, positions=2048, salt=3),
        # the tokens of a large prefill step on the 8B shape, f32 projections into a bf16 cache, last rows of the batch unused
        dict(name="append-8000-bf16", kind="append", tokens=8000, pad=192, H=32, KV=8, hd=128, rot=128, src="f32", dtype="bf16", page=16, positions=8192, salt=4),
        # the smallest attention: one request of the 135M shape, 260 cached positions, f32
        dict(name="attn-1x260-f32", kind="attention", mode="steps", R=1, fresh=1, least=260, most=260, H=9, KV=3, hd=64, dtype="f32", page=16, window=0, pad=0, salt=5),
        # a serving batch on the 8B shape: lengths from a few to four thousand, one new token each
        dict(name="attn-64-steps-bf16", kind="attention", mode="steps", R=64, fresh=1, least=64, most=4096, H=32, KV=8, hd=128, dtype="bf16", page=16, window=0, pad=0, salt=6),
        # one user deep in a long document
        dict(name="attn-1x32000-f16", kind="attention", mode="steps", R=1, fresh=1, least=32000, most=32000, H=32, KV=8, hd=128, dtype="f16", page=64, window=0, pad=0, salt=7),
        # drafts of five tokens checked at once in f32, heads without sharing, a sliding window
        dict(name="attn-24x5-f32-window", kind="attention", mode="few", R=24, fresh=5, least=100, most=3000, H=12, KV=12, hd=64, dtype="f32", page=16, window=1000, pad=7, salt=8),
        # a chunk of a long prompt while nothing else waits
        dict(name="attn-chunk-500-bf16", kind="attention", mode="few", R=1, fresh=500, least=8192, most=8192, H=32, KV=8, hd=128, dtype="bf16", page=16, window=0, pad=12, salt=9),
        # a mixed step of the 1.1B shape: three prompts' chunks beside decoding requests
        dict(name="attn-mixed-f16", kind="attention", mode="mixed", R=24, fresh=600, least=30, most=2000, H=32, KV=4, hd=64, dtype="f16", page=32, window=0, pad=0, salt=10),
        # a whole prompt on the 1.1B shape in f32, the type that the framework's models compute in
        dict(name="attn-prompt-1000-f32", kind="attention", mode="few", R=1, fresh=1000, least=0, most=0, H=32, KV=4, hd=64, dtype="f32", page=16, window=0, pad=0, salt=11),
        # four prompts of two thousand tokens at once: time to the first token of a busy server
        dict(name="attn-4x2000-bf16", kind="attention", mode="few", R=4, fresh=2000, least=0, most=0, H=32, KV=8, hd=128, dtype="bf16", page=16, window=0, pad=0, salt=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind, salt = rng.choice(["plan", "append", "attention", "attention", "attention", "attention"]), rng.randint(100, 1 << 30)
    page = rng.choice([16, 16, 32, 64, 128, 256])
    if kind == "plan":
        R = _log(rng, 1, 4000)
        return dict(kind=kind, R=R, fresh=_log(rng, 1, 2000), prompts=rng.randint(0, min(R, 40)), ended=rng.randint(0, R // 8), most=_log(rng, 32, 8000), page=page, pad=rng.choice([0, 0, 77, 1000]), salt=salt)
    H, KV, hd = rng.choice(HEADS)
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    if kind == "append":
        return dict(kind=kind, tokens=_log(rng, 1, 8000 * 48 * 128 // ((H + 2 * KV) * max(hd, 128))), pad=rng.choice([0, 0, 3, 100]), H=H, KV=KV, hd=hd, rot=rng.choice([hd, hd, hd, hd // 2 // 8 * 8, 0]),
                    src=rng.choice(["f32", dtype]), dtype=dtype, page=page, positions=_log(rng, 256, 16384), salt=salt)
    window = 0 if rng.random() < 0.7 else _log(rng, 8, 4000)
    mode = rng.choice(["steps", "steps", "few", "few", "mixed"])
    most_keys = 250 * 1000 * 1000 // (KV * hd * _BYTES[dtype])  # over all requests: half a gigabyte of keys and values
    most_pairs = 8 * 1000 * 1000 * 4096 // (H * hd)  # over all requests, padded to the longest
    if mode == "steps":
        R = _log(rng, 1, 128)
        fresh, most = 1, _log(rng, 1, min(32000, most_keys // R))
        least = rng.choice([most, max(0, most // 50)])
    elif mode == "few":
        fresh = _log(rng, 2, 2000)
        R = _log(rng, 1, max(1, 4000 // fresh) if fresh > 16 else 64)
        most = rng.choice([0, _log(rng, 1, 8000)])
        most = min(most, max(0, most_pairs // (R * fresh) - fresh), most_keys // R)
        least = rng.choice([most, most // 3])
    else:
        R, fresh, most = _log(rng, 4, 48), _log(rng, 32, 600), _log(rng, 30, 3000)
        most = min(most, max(30, most_pairs // (R * fresh) - fresh), most_keys // R)
        least = most // 20
    return dict(kind=kind, mode=mode, R=R, fresh=fresh, least=least, most=most, H=H, KV=KV, hd=hd, dtype=dtype, page=page, window=window, pad=rng.choice([0, 0, 5]), salt=salt)


# ---- lengths (from the case alone) ------------------------------------------------------------------------------------


def _lengths(case):
    """(cached, fresh) per request, as int64 arrays."""
    r = np.random.RandomState(case["salt"] % (1 << 31))
    R = case["R"]
    if case["kind"] == "plan":
        cached = np.exp(r.uniform(0, math.log(case["most"] + 1), R)).astype(np.int64)
        fresh = np.ones(R, np.int64)
        order = r.permutation(R)
        with_prompt, ended = order[:case["prompts"]], order[R - case["ended"]:] if case["ended"] else order[:0]
        cached[with_prompt] = r.randint(0, 2, len(with_prompt)) * cached[with_prompt]
        fresh[with_prompt] = np.maximum(1, (r.rand(len(with_prompt)) * case["fresh"]).astype(np.int64))
        fresh[ended] = -1
        return cached, fresh
    cached = r.randint(case["least"], case["most"] + 1, R).astype(np.int64)
    fresh = np.full(R, case["fresh"], np.int64)
    if case["mode"] == "mixed":  # every eighth brings a chunk, the others a token
        fresh = np.where(np.arange(R) % 8 == 0, np.maximum(1, (case["fresh"] * (0.5 + 0.5 * r.rand(R))).astype(np.int64)), 1)
    return cached, fresh


def _up(a, b):
    return -(-a // b)


def _visible(case):
    """Pairs of a new token and a key that it sees, and the keys that any token of a request sees, over all requests."""
    cached, fresh = _lengths(case)
    pairs = keys = 0
    for c, f in zip(cached.tolist(), fresh.tolist()):
        p = np.arange(c, c + f, dtype=np.int64) + 1
        seen = p if not case["window"] else np.minimum(p, case["window"])
        pairs += int(seen.sum())
        keys += c + f - max(0, c + 1 - (case["window"] or c + f + 1))
    return pairs, keys


def work(case):
    if case["kind"] == "plan":
        cached, fresh = _lengths(case)
        n, held = np.maximum(fresh, 0), _up(cached, case["page"])
        need = np.where(fresh >= 0, _up(cached + n, case["page"]) - held, 0).sum()
        tokens = int(n.sum()) + case["pad"]
        back = np.where(fresh < 0, held, 0).sum()
        return {"bytes": 4.0 * (3 * case["R"] + 2 * tokens + np.minimum(n, 1).sum() + 2 * need + 2 * back), "flops": 0.0}
    if case["kind"] == "append":
        each = (case["H"] + 2 * case["KV"]) * case["hd"]
        table = min(case["tokens"], case["positions"]) * case["rot"] * 4.0
        return {"bytes": case["tokens"] * (each * (_BYTES[case["src"]] + _BYTES[case["dtype"]]) + 8.0) + table, "flops": case["tokens"] * 3.0 * (case["H"] + case["KV"]) * case["rot"]}
    pairs, keys = _visible(case)
    tokens = int(_lengths(case)[1].sum())
    b = _BYTES[case["dtype"]]
    return {"bytes": b * (2.0 * case["KV"] * case["hd"] * keys + 2.0 * tokens * case["H"] * case["hd"]) + 4.0 * keys / case["page"], "flops": 4.0 * case["H"] * case["hd"] * pairs}


# ---- inputs -------------------------------------------------------------------------------------------------------------


def _gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + salt) % (1 << 62))


def _normal(seed, salt, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=_gen(seed, salt), device="cuda") * std).to(_TORCH[dtype])


def _int(a):
    return torch.as_tensor(np.asarray(a), device="cuda").to(torch.int32)


def _pool(case, seed, held, spare):
    """Pages of every request in an order of the seed's, and the free ones: (table, ring, pages)."""
    total = int(held.sum())
    pages = total + spare
    order = np.random.RandomState((int(seed) * 7919 + 5) % (1 << 31)).permutation(pages).astype(np.int32)
    return order[:total], order[total:], pages


def _table(held, flat, width):
    table = np.full((len(held), width), -1, np.int32)
    at = np.arange(width)[None, :] < held[:, None]
    table[at] = flat
    return table


def _rope(case):
    half = case["rot"] // 2
    inv = 10000.0 ** (-2.0 * torch.arange(half, device="cuda", dtype=torch.float64) / max(case["rot"], 1))
    a = torch.arange(case["positions"], device="cuda", dtype=torch.float64)[:, None] * inv[None, :]
    return torch.stack([a.cos(), a.sin()], -1).float()


def _inputs(case, seed):
    """Torch tensors of a case, by name."""
    seed = int(seed) % (1 << 31)
    page = case["page"]
    if case["kind"] == "plan":
        cached, fresh = _lengths(case)
        held, n = _up(cached, page), np.maximum(fresh, 0)
        need = int(np.where(fresh >= 0, _up(cached + n, page) - held, 0).sum())
        flat, free, pages = _pool(case, seed, held, need + 100)
        first = np.random.RandomState(seed).randint(pages)
        ring = np.full(pages, -1, np.int32)
        ring[(first + np.arange(len(free))) % pages] = free
        return dict(cached=_int(cached), fresh=_int(fresh), table=_int(_table(held, flat, int(_up(cached + n, page).max()) + 2)), ring=_int(ring), words=_int([first, len(free), 0]))
    if case["kind"] == "append":
        T, H, KV, hd = case["tokens"] + case["pad"], case["H"], case["KV"], case["hd"]
        pages = _up(case["tokens"], page) + 7
        r = np.random.RandomState(seed)
        slots, positions = np.full(T, -1, np.int64), np.full(T, -1, np.int64)
        slots[:case["tokens"]] = r.permutation(pages * page)[:case["tokens"]]
        positions[:case["tokens"]] = (r.randint(case["positions"]) + np.arange(case["tokens"])) % case["positions"]
        kv = (pages, KV, page, hd)
        made = dict(qkv=_normal(seed, 1, (T, (H + 2 * KV) * hd), case["src"]), positions=_int(positions), slots=_int(slots), k=_normal(seed, 2, kv, case["dtype"]), v=_normal(seed, 3, kv, case["dtype"]))
        if case["rot"]:
            made["rope"] = _rope(case)
        return made
    cached, fresh = _lengths(case)
    held = _up(cached + fresh, page)
    flat, _, pages = _pool(case, seed, held, 9)
    tokens = int(fresh.sum()) + case["pad"]
    kv = (pages, case["KV"], page, case["hd"])
    # scores spread over several units: a row's softmax is neither flat nor one key
    k = _normal(seed, 2, kv, case["dtype"], 1.5)
    return dict(q=_normal(seed, 1, (tokens, case["H"], case["hd"]), case["dtype"], 1.5), k=k, v=_normal(seed, 3, kv, case["dtype"]), table=_int(_table(held, flat, int(held.max()) + 1)),
                cached=_int(cached), starts=_int(np.concatenate([[0], np.cumsum(fresh)])))


class _Memory:
    """A device tensor of the library as torch sees it, without a copy."""

    def __init__(self, t):
        self.t = t
        self.__cuda_array_interface__ = {"shape": t.shape, "typestr": t.np_dtype.str, "data": (t.ptr.value, False), "version": 2}


def _view(t):
    v = torch.as_tensor(_Memory(t), device="cuda")
    return v.view(torch.bfloat16) if t.rdtype == nn.BF16 else v


def _tensor(dev, shape, dtype):
    return nn.Tensor(dev, shape, np.int32) if dtype == "i32" else nn.Tensor(dev, shape, _NP[dtype], _DTYPE[dtype])


_NAMES = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16", torch.int32: "i32"}


def prepare(case, seed):
    dev = nn.Device.cuda(0)
    t, v = {}, {}
    for name, x in _inputs(case, seed).items():
        t[name] = _tensor(dev, x.shape, _NAMES[x.dtype])
        v[name] = _view(t[name])
        v[name].copy_(x)
    # what a serving loop keeps from step to step: the buffers that the calls write
    cached, fresh = _lengths(case) if case["kind"] != "append" else (None, None)
    if case["kind"] == "plan":
        T = int(np.maximum(fresh, 0).sum()) + case["pad"]
        made = {"starts": (case["R"] + 1,), "positions": (T,), "slots": (T,), "words_out": (3,)}
        t.update({n: _tensor(dev, s, "i32") for n, s in made.items()})
    elif case["kind"] == "append":
        t["out"] = _tensor(dev, (case["tokens"] + case["pad"], case["H"], case["hd"]), case["dtype"])
    else:
        t["out"] = _tensor(dev, t["q"].shape, case["dtype"])
    for name in t:
        if name not in v:
            v[name] = _view(t[name])
            v[name].zero_()
    torch.cuda.synchronize()
    most = dict(most_fresh=int(fresh.max()), most_len=int((cached + fresh).max()), total=int(fresh.sum())) if case["kind"] == "attention" else {}
    return dict(kind=case["kind"], case=dict(case), t=t, v=v, **most)


# ---- passes ------------------------------------------------------------------------------------------------------------


def _plan_outputs(v):
    return {n: v[n] for n in ("table", "ring", "starts", "positions", "slots", "words_out")}


def run(state):
    case, t, v = state["case"], state["t"], state["v"]
    if state["kind"] == "plan":
        if own:
            nn.page_plan(t["cached"], t["fresh"], t["table"], t["ring"], t["words"], case["page"], out=nn.PagePlan(t["starts"], t["positions"], t["slots"], t["words_out"]))
        else:
            _plan(case, v)
        return _plan_outputs(v)
    if state["kind"] == "append":
        if own:
            nn.paged_append(t["qkv"], t["positions"], t["slots"], t["k"], t["v"], rope=t.get("rope"), out=t["out"])
        else:
            _append(case, v)
        return v["out"], v["k"], v["v"]
    if own:
        nn.paged_attention(t["q"], t["k"], t["v"], t["table"], t["cached"], t["starts"], state["most_fresh"], state["most_len"], window=case["window"], out=t["out"])
    else:
        _attention(case, v, state["most_fresh"], state["most_len"], state["total"])
    return v["out"]


def _exclusive(n):
    return torch.cat([torch.zeros(1, dtype=torch.int64, device=n.device), n.cumsum(0)])


def _plan(case, v):
    page, pages = case["page"], v["ring"].numel()
    cached, fresh, table, ring = v["cached"].long(), v["fresh"].long(), v["table"], v["ring"]
    first, free = v["words"][0].long(), v["words"][1].long()
    n, held = fresh.clamp(min=0), (cached + page - 1) // page
    need = torch.where(fresh >= 0, (cached + n + page - 1) // page - held, 0)
    back = torch.where(fresh < 0, held, 0)
    starts, needs, backs = _exclusive(n), _exclusive(need), _exclusive(back)
    # new pages: the ring's next ones, in the order of the requests
    j = torch.arange(table.shape[1], device=table.device)[None, :] - held[:, None]
    new = (j >= 0) & (j < need[:, None])
    taken = torch.where(new, ring[(first + needs[:-1, None] + j) % pages], table)
    # pages of ended requests: behind the free ones
    o = (torch.arange(pages, device=ring.device) - first - free) % pages
    row = torch.searchsorted(backs[1:], o, right=True).clamp(max=len(cached) - 1)
    returned = table[row, (o - backs[row]).clamp(0, table.shape[1] - 1)]
    v["ring"].copy_(torch.where(o < backs[-1], returned, ring))
    v["table"].copy_(taken)
    t = torch.arange(v["slots"].numel(), device=ring.device)
    row = torch.searchsorted(starts[1:], t, right=True).clamp(max=len(cached) - 1)
    used = t < starts[-1]
    pos = cached[row] + t - starts[row]
    v["positions"].copy_(torch.where(used, pos, -1))
    v["slots"].copy_(torch.where(used, taken.long()[row, (pos // page).clamp(0, table.shape[1] - 1)] * page + pos % page, -1))
    v["starts"].copy_(starts)
    v["words_out"].copy_(torch.stack([(first + needs[-1]) % pages, free - needs[-1] + backs[-1], torch.zeros_like(first)]))


def _append(case, v):
    T, H, KV, hd, page, half = case["tokens"], case["H"], case["KV"], case["hd"], case["page"], case["rot"] // 2
    x = v["qkv"][:T].float().view(T, H + 2 * KV, hd)
    slots = v["slots"][:T].long()
    if half:
        cs = v["rope"][v["positions"][:T].long()][:, None]
        c, s = cs[..., 0], cs[..., 1]
        a, b = x[:, :H + KV, :half], x[:, :H + KV, half:2 * half]
        x = torch.cat([torch.cat([a * c - b * s, b * c + a * s, x[:, :H + KV, 2 * half:]], -1), x[:, H + KV:]], 1)
    x = x.to(v["k"].dtype)
    v["out"][:T] = x[:, :H]
    v["k"][slots // page, :, slots % page] = x[:, H:H + KV]
    v["v"][slots // page, :, slots % page] = x[:, H + KV:]


def _attention(case, v, most_fresh, most_len, total):
    R, H, KV, hd, page = case["R"], case["H"], case["KV"], case["hd"], case["page"]
    n, rep = -(-most_len // page), H // KV
    table, cached, starts = v["table"][:, :n].long().clamp(min=0), v["cached"].long(), v["starts"].long()
    i = torch.arange(most_fresh, device=table.device)
    length = cached + starts[1:] - starts[:-1]
    key = torch.arange(n * page, device=table.device)

    def gathered(pool):
        x = pool[table].float().permute(0, 2, 1, 3, 4).reshape(R, KV, n * page, hd)
        return x * (key < length[:, None])[:, None, :, None]

    at = (starts[:-1, None] + i).clamp(max=v["q"].shape[0] - 1)
    q = v["q"][at].float().view(R, most_fresh, KV, rep, hd).permute(0, 2, 3, 1, 4).reshape(R, KV, rep * most_fresh, hd)
    s = (q @ gathered(v["k"]).transpose(-1, -2)).view(R, KV, rep, most_fresh, n * page) * (1.0 / math.sqrt(hd))
    pos = cached[:, None] + i
    seen = key <= pos[..., None]
    if case["window"]:
        seen = seen & (key > pos[..., None] - case["window"])
    s = torch.where(seen[:, None, None], s, -math.inf)
    s = torch.exp(s - s.amax(-1, keepdim=True))
    s = s / s.sum(-1, keepdim=True)
    o = (s.view(R, KV, rep * most_fresh, n * page) @ gathered(v["v"])).view(R, KV, rep, most_fresh, hd).permute(0, 3, 1, 2, 4).reshape(R, most_fresh, H, hd)
    t = torch.arange(total, device=table.device)
    row = torch.searchsorted(starts[1:], t, right=True)
    v["out"][:total] = o[row, t - starts[row]].to(v["out"].dtype)


# ---- the same from the definition, in 64 bits ------------------------------------------------------------------------------


def exact(case, seed):
    x = _inputs(case, seed)
    page = case["page"]
    if case["kind"] == "plan":
        return None  # whole numbers: they have to be equal
    if case["kind"] == "append":
        T, H, KV, hd, half = case["tokens"], case["H"], case["KV"], case["hd"], case["rot"] // 2
        y = x["qkv"].double().reshape(-1, H + 2 * KV, hd)
        if half:
            z = torch.view_as_complex(torch.stack([y[:T, :H + KV, :half], y[:T, :H + KV, half:2 * half]], -1).contiguous())
            z = z * torch.view_as_complex(x["rope"].double())[x["positions"][:T].long()][:, None]
            y[:T, :H + KV, :half], y[:T, :H + KV, half:2 * half] = z.real, z.imag
        out = torch.zeros((T + case["pad"], H, hd), dtype=torch.float64, device="cuda")
        out[:T] = y[:T, :H]
        pools = []
        for pool, part in ((x["k"], y[:T, H:H + KV]), (x["v"], y[:T, H + KV:])):
            flat = pool.double().transpose(1, 2).reshape(-1, KV, hd)
            flat[x["slots"][:T].long()] = part
            pools.append(flat.view(-1, page, KV, hd).transpose(1, 2).contiguous())
        return out, pools[0], pools[1]
    pairs, keys = _visible(case)
    if pairs * case["H"] * case["hd"] > 4e12:
        return None
    cached, fresh = _lengths(case)
    out = torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")
    t0 = 0
    for r, (c, f) in enumerate(zip(cached.tolist(), fresh.tolist())):
        pages = x["table"][r, :_up(c + f, page)].long()
        k, val = (x[n][pages].double().transpose(0, 1).reshape(case["KV"], -1, case["hd"])[:, :c + f] for n in ("k", "v"))
        for a in range(0, f, 256):
            rows = torch.arange(a, min(a + 256, f), device="cuda")
            low = max(0, c + a + 1 - case["window"]) if case["window"] else 0
            high = c + int(rows[-1]) + 1
            far = c + rows[:, None] - torch.arange(low, high, device="cuda")
            hidden = (far < 0) | (far >= case["window"]) if case["window"] else far < 0
            q = x["q"][t0 + rows].double().reshape(len(rows), case["KV"], -1, case["hd"])
            s = torch.einsum("tghd,gkd->ghtk", q, k[:, low:high]) / math.sqrt(case["hd"])
            s = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
            out[t0 + rows] = torch.einsum("ghtk,gkd->tghd", s, val[:, low:high]).reshape(len(rows), case["H"], case["hd"])
        t0 += f
    return out
