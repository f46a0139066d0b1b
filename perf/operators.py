"""The operators that read and shorten a live KV cache, as cases that can be
timed and compared: attention over a 16- or 32-bit cache with a sliding window
and first tokens that stay visible, the same over a cache held in 4 bits, the
store and load of that cache, and eviction by accumulated attention weight.

listed() are the cases, draw() one more of the same ranges, prepare() what a
serving program has in hand before the call, run() one pass, work() what a pass
cannot do without, exact() the same results in 64 bits.  own = False computes
the plain form in elementary torch operations, own = True makes the calls a
user makes.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
BLOCK = 32                 # values that share one scale in the 4-bit cache


def listed():
    return [
        # one new token of a short conversation, one agent, one layer of the
        # 32-head, head_dim-64 shape: the call where latency is everything
        dict(name="decode_short", kind="attend", dtype="bf16", copies=1, heads=32, group=1, dim=64, tokens=1024,
             least=577, rows=1, ragged=False, window=0, sinks=0, weights=False),
        # one new token of each of the 8 agents over the rehydrated f32 pool of
        # 1,024 tokens, ragged
        dict(name="decode_agents", kind="attend", dtype="f32", copies=8, heads=32, group=1, dim=64, tokens=1024,
             least=828, rows=1, ragged=False, window=0, sinks=0, weights=False),
        # one new token over long contexts at head_dim 128, four query heads to
        # a KV head, with the weights that a later eviction goes by
        dict(name="decode_long", kind="attend", dtype="bf16", copies=4, heads=8, group=4, dim=128, tokens=32768,
             least=30011, rows=1, ragged=False, window=0, sinks=0, weights=True),
        # a whole prompt of 8,192 tokens, causal: the largest call
        dict(name="prompt", kind="attend", dtype="bf16", copies=1, heads=8, group=4, dim=128, tokens=8192,
             least=8192, rows=8192, ragged=False, window=0, sinks=0, weights=False),
        # a padded batch of prompt chunks behind caches of other lengths, a
        # window of 1,024 with 4 first tokens visible, weights accumulated
        dict(name="chunk_window", kind="attend", dtype="f16", copies=3, heads=8, group=3, dim=64, tokens=6000,
             least=2500, rows=701, ragged=True, window=1024, sinks=4, weights=True),
        # one new token of each of 8 agents over 4-bit caches, 16-bit queries
        dict(name="decode4_agents", kind="attend4", dtype="f16", copies=8, heads=32, group=1, dim=64, tokens=1024,
             least=828, rows=1, ragged=False, window=0, sinks=0, weights=False),
        # the long contexts again, held in 4 bits
        dict(name="decode4_long", kind="attend4", dtype="bf16", copies=4, heads=8, group=4, dim=128, tokens=32768,
             least=30011, rows=1, ragged=False, window=0, sinks=0, weights=False),
        # chunks of a prompt over 4-bit caches with window and first tokens
        dict(name="chunk4_window", kind="attend4", dtype="bf16", copies=2, heads=8, group=4, dim=128, tokens=12000,
             least=9001, rows=513, ragged=True, window=4096, sinks=8, weights=True),
        # one new token of every agent and layer put into the 4-bit cache and
        # read back: the smallest store
        dict(name="store4_token", kind="store4", dtype="bf16", copies=8, layers=24, heads=32, dim=64, tokens=1024,
             rows=1),
        # a rehydrated f32 pool of 1,024 tokens moved into the 4-bit cache and
        # read back
        dict(name="store4_pool", kind="store4", dtype="f32", copies=1, layers=24, heads=32, dim=64, tokens=1024,
             rows=1024),
        # the caches of 8 agents halved
        dict(name="evict_agents", kind="evict", dtype="bf16", copies=8, layers=1, heads=32, dim=64, tokens=1024,
             least=828, budget=512, sinks=4, recent=100, coarse=False),
        # long contexts of 8 layers cut to a quarter; many equal weights
        dict(name="evict_long", kind="evict", dtype="bf16", copies=1, layers=8, heads=8, dim=128, tokens=32768,
             least=32001, budget=8192, sinks=16, recent=1024, coarse=True),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend4", "attend4", "store4", "evict"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    dim = rng.choice([64, 128])
    if kind in ("attend", "attend4"):
        copies, heads = rng.randint(1, 8), rng.randint(1, 16)
        group = rng.randint(1, 8)
        form = rng.choice(["token", "few", "chunk"])
        rows = 1 if form == "token" else rng.randint(2, 16) if form == "few" else _log(rng, 17, 2048)
        tokens = max(_log(rng, 16, 32768), rows)
        if dtype == "f32":
            rows = min(rows, 700)
        # the plain form holds every logit: bound them, and the cache's size
        while copies * heads * group * rows * tokens > 1 << 29 or copies * heads * tokens * dim > 1 << 28:
            if copies > 1:
                copies -= 1
            elif heads > 1:
                heads -= 1
            else:
                tokens = max(rows, tokens // 2)
                group = max(1, group // 2)
        window = rng.choice([0, 0, _log(rng, 1, 8192)])
        return dict(kind=kind, dtype=dtype, copies=copies, heads=heads, group=group, dim=dim, tokens=tokens,
                    least=rng.randint(max(1, tokens // 2), tokens), rows=rows, ragged=rng.random() < 0.5,
                    window=window, sinks=rng.choice([0, 1, 4, 17]) if window else 0, weights=rng.random() < 0.5)
    copies, layers, heads = rng.randint(1, 4), rng.randint(1, 8), rng.randint(1, 32)
    tokens = _log(rng, 8, 32768)
    while copies * layers * heads * tokens * dim > 1 << 26:
        tokens //= 2
    if kind == "store4":
        return dict(kind=kind, dtype=dtype, copies=copies, layers=layers, heads=heads, dim=dim, tokens=tokens,
                    rows=_log(rng, 1, tokens))
    budget = rng.randint(1, tokens)
    sinks = rng.randint(0, min(16, budget))
    return dict(kind=kind, dtype=dtype, copies=copies, layers=layers, heads=heads, dim=dim, tokens=tokens,
                least=rng.randint(1, tokens), budget=budget, sinks=sinks,
                recent=rng.randint(0, (budget - sinks) // 2), coarse=rng.random() < 0.5)


# ---------------------------------------------------------------- inputs
def _gen(seed, device="cuda"):
    g = torch.Generator(device=device)
    g.manual_seed(int(seed))
    return g


def _lens(case, g):
    """Lengths between `least` and the capacity; the first copy is full."""
    n = torch.randint(case["least"], case["tokens"] + 1, (case["copies"],), generator=g, device="cuda")
    n[0] = case["tokens"]
    return n.to(torch.int32)


def _cache(case, layers, g):
    """Keys with per-channel scales and a few large channels, values Gaussian:
    f32 [copies, layers, 2 (K|V), heads, tokens, dim]."""
    D = case["dim"]
    x = torch.randn((case["copies"], layers, 2, case["heads"], case["tokens"], D), generator=g, device="cuda")
    scale = torch.exp(0.3 * torch.randn((case["heads"], 1, D), generator=g, device="cuda"))
    outlier = torch.rand((case["heads"], 1, D), generator=g, device="cuda") < 0.03
    x[:, :, 0] *= torch.where(outlier, scale * 3.0, scale)
    return x


def prepare(case, seed):
    g = _gen(seed)
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    C, H, D, T = case["copies"], case["heads"], case["dim"], case["tokens"]
    s = dict(case=dict(case), kind=kind)
    if kind in ("attend", "attend4"):
        x = _cache(case, 1, g)
        s["lens"] = _lens(case, g)
        n = case["rows"]
        s["q"] = torch.randn((C, n, H * case["group"], D), generator=g, device="cuda").to(dt)
        s["q_lens"] = None
        if case["ragged"]:
            ql = torch.randint(max(1, n // 2), n + 1, (C,), generator=g, device="cuda")
            ql[0] = n
            s["q_lens"] = ql.to(torch.int32)
        # rows behind a copy's last are not written: the caller's buffer holds zeros there
        s["out"] = torch.zeros_like(s["q"])
        # what earlier passes of this size left on each slot, on average
        s["weights"] = None
        if case["weights"]:
            s["weights"] = torch.rand((C, H, T), generator=g, device="cuda") * (2.0 * n * case["group"] / T)
        if kind == "attend":
            s["buf"] = x.to(dt)
        else:
            s["codes"], s["scales"] = _quantise(x)
        del x
    elif kind == "store4":
        n = case["rows"]
        x = _cache(dict(case, tokens=n), case["layers"], g)
        s["keys"], s["values"] = x[:, :, 0].to(dt).contiguous(), x[:, :, 1].to(dt).contiguous()
        del x
        s["first"] = torch.randint(0, T - n + 1, (C,), generator=g, device="cuda").to(torch.int32)
        shape = (C, case["layers"], 2, H, T)
        s["codes"] = torch.zeros((*shape, D // 2), dtype=torch.uint8, device="cuda")
        s["scales"] = torch.zeros((*shape, D // BLOCK), dtype=torch.uint8, device="cuda")
    else:
        s["buf"] = _cache(case, case["layers"], g).to(dt)
        s["lens"] = _lens(case, g)
        # a few keys hold most of the weight; `coarse` rounds it so that many are equal
        w = torch.rand((C, case["layers"], H, T), generator=g, device="cuda").pow(8) * 100.0
        s["weights"] = torch.floor(w) if case["coarse"] else w
    if own:
        from provekv_amd.pool import DeviceKVCache, FourBitKVCache
        layers = case.get("layers", 1)
        if kind in ("attend4", "store4"):
            s["cache"] = FourBitKVCache.over(s["codes"], s["scales"])
        else:
            s["cache"] = DeviceKVCache.over(s["buf"])
        if kind == "evict":
            s["into"] = DeviceKVCache(layers, H, case["budget"], D, dtype=dt, copies=C)
    return s


# ---------------------------------------------------------------- plain forms
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _quantise(x):
    """4-bit codes (two a byte, the even element low) and scale bytes of f32
    rows [..., dim]: blocks of 32, the smallest scale 2^e with
    max |x| <= 7 * 2^e; a value goes to the nearest of GRID, half way to the
    even code."""
    b = x.reshape(*x.shape[:-1], -1, BLOCK).double()
    m, e = torch.frexp(b.abs().amax(dim=-1))
    e = (e - 3 + (m > 0.875).to(e.dtype)).clamp(-125, 125)
    e = torch.where(m == 0, torch.full_like(e, -125), e)
    y = torch.ldexp(b, -e.unsqueeze(-1))
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75).to(torch.uint8) + (a > 1.25).to(torch.uint8)
            + (a >= 1.75).to(torch.uint8) + (a > 2.5).to(torch.uint8) + (a >= 3.5).to(torch.uint8)
            + (a > 5.0).to(torch.uint8))
    code = code + torch.signbit(y).to(torch.uint8) * 8
    code = code.reshape(*x.shape[:-1], -1, 2)
    return code[..., 0] + 16 * code[..., 1], (e + 127).to(torch.uint8)


def _values(codes, scales):
    """The f32 values that codes and scale bytes stand for."""
    c = torch.stack((codes & 15, codes >> 4), dim=-1).reshape(*codes.shape[:-1], -1, BLOCK).long()
    grid = torch.tensor(GRID, dtype=torch.float32, device=codes.device)
    v = grid[c & 7] * (1.0 - 2.0 * (c >> 3).float())
    v = torch.ldexp(v, scales.int().unsqueeze(-1) - 127)
    return v.reshape(*codes.shape[:-1], -1)


def _plain_attend(s, k, v):
    """k, v: [copies, heads, tokens, dim] f32."""
    case, q, lens = s["case"], s["q"], s["lens"]
    C, n, Hq, D = q.shape
    H, T, G = case["heads"], case["tokens"], case["group"]
    ql = s["q_lens"] if s["q_lens"] is not None else torch.full_like(lens, n)
    rows = torch.arange(n, device=q.device)
    pos = (lens - ql).view(C, 1, 1) + rows.view(1, n, 1)
    slot = torch.arange(T, device=q.device).view(1, 1, T)
    see = slot <= pos
    if case["window"]:
        see = see & ((pos - slot < case["window"]) | (slot < case["sinks"]))
    real = rows.view(1, n) < ql.view(C, 1)
    see = (see & real.view(C, n, 1)).view(C, 1, n, 1, T)
    x = q.float().reshape(C, n, H, G, D).permute(0, 2, 1, 3, 4).reshape(C, H, n * G, D)
    logit = torch.matmul(x, k.transpose(-1, -2)).view(C, H, n, G, T) * (1.0 / math.sqrt(D))
    logit = logit.masked_fill(~see, -math.inf)
    top = logit.amax(dim=-1, keepdim=True)
    p = torch.exp(logit - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(dim=-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    del logit
    o = torch.matmul(p.view(C, H, n * G, T), v)
    o = o.view(C, H, n, G, D).permute(0, 2, 1, 3, 4).reshape(C, n, Hq, D).to(q.dtype)
    o = torch.where(real.view(C, n, 1, 1), o, s["out"])
    if s["weights"] is None:
        return {"out": o}
    s["weights"] += p.sum(dim=(2, 3))
    return {"out": o, "weights": s["weights"]}


def _plain_evict(s):
    case, lens, w = s["case"], s["lens"], s["weights"]
    C, L, H, T = w.shape
    B = case["budget"]
    slot = torch.arange(T, device=w.device).view(1, 1, 1, T)
    n = lens.view(C, 1, 1, 1)
    # order of giving up: everything behind the length last of all, then the
    # lightest; kept without question: the first and the last slots
    key = torch.where((slot < case["sinks"]) | (slot >= n - case["recent"]), torch.full_like(w, math.inf), w)
    key = torch.where(slot < n, key, torch.full_like(w, -math.inf))
    best = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :B]
    best = torch.where(best < n, best, torch.full_like(best, T))
    best = torch.sort(best, dim=-1).values
    there = best < n
    at = torch.where(there, best, torch.zeros_like(best))
    buf = s["buf"].permute(0, 1, 3, 4, 2, 5)                        # [C, L, H, T, 2, D]
    take = at.view(C, L, H, B, 1, 1).expand(C, L, H, B, 2, buf.shape[-1])
    rows = torch.gather(buf, 3, take)
    rows = torch.where(there.view(C, L, H, B, 1, 1), rows, torch.zeros_like(rows))
    kept_w = torch.where(there, torch.gather(w, 3, at), torch.zeros((), device=w.device))
    kept = torch.where(there, best, torch.full_like(best, -1)).to(torch.int32)
    return {"buf": rows.permute(0, 1, 4, 2, 3, 5).contiguous(), "weights": kept_w, "kept": kept,
            "lens": torch.clamp(lens, max=B)}


def _plain_store(s):
    C, L, H, n, D = s["keys"].shape
    at = s["first"].long().view(C, 1, 1, 1, 1, 1) + torch.arange(n, device="cuda").view(1, 1, 1, 1, n, 1)
    rows = torch.stack((s["keys"], s["values"]), dim=2).float()
    codes, scales = _quantise(rows)
    at_c, at_s = at.expand(codes.shape), at.expand(scales.shape)
    s["codes"].scatter_(4, at_c, codes)
    s["scales"].scatter_(4, at_s, scales)
    v = _values(torch.gather(s["codes"], 4, at_c), torch.gather(s["scales"], 4, at_s)).to(s["keys"].dtype)
    return {"keys": v[:, :, 0], "values": v[:, :, 1]}


def run(state):
    case, kind = state["case"], state["kind"]
    if own:
        if kind in ("attend", "attend4"):
            out = state["cache"].attend(0, state["q"], state["lens"], q_lens=state["q_lens"], window=case["window"],
                                        sinks=case["sinks"], weights=state["weights"], out=state["out"])
            return {"out": out} if state["weights"] is None else {"out": out, "weights": state["weights"]}
        if kind == "store4":
            state["cache"].store(state["keys"], state["values"], state["first"])
            keys, values = state["cache"].load(state["first"], case["rows"], dtype=state["keys"].dtype)
            return {"keys": keys, "values": values}
        into = state["into"]
        kept, lens, weights = state["cache"].evict(state["lens"], state["weights"], case["budget"],
                                                   sinks=case["sinks"], recent=case["recent"], into=into)
        return {"buf": into.buf, "weights": weights, "kept": kept, "lens": lens}
    if kind == "attend":
        return _plain_attend(state, state["buf"][:, 0, 0].float(), state["buf"][:, 0, 1].float())
    if kind == "attend4":
        x = _values(state["codes"][:, 0], state["scales"][:, 0])
        return _plain_attend(state, x[:, 0], x[:, 1])
    if kind == "store4":
        return _plain_store(state)
    return _plain_evict(state)


# ---------------------------------------------------------------- work
def _seen(case):
    """(visible (row, slot) pairs of one copy and head, visible slots) at the
    expected length and rows, or the exact ones where they are given."""
    n = (case["least"] + case["tokens"]) // 2
    rows = case["rows"] if not case["ragged"] else (case["rows"] + max(1, case["rows"] // 2)) // 2
    pairs, reach = 0, 0
    w, k = case["window"], case["sinks"]
    for i in range(rows):
        p = n - rows + i + 1                   # slots up to and with the row's own
        if p <= 0:
            continue
        low = max(0, p - w) if w else 0
        pairs += p - low + min(k, low)
        if reach == 0:
            reach = -low + min(k, low)         # from the first row's window on
    return pairs, max(1, reach + n)


def work(case):
    C, H, D = case["copies"], case["heads"], case["dim"]
    e = BYTES[case["dtype"]]
    row4 = D / 2 + D / BLOCK
    if case["kind"] in ("attend", "attend4"):
        pairs, slots = _seen(case)
        G = case["group"]
        rows = case["rows"] if not case["ragged"] else (case["rows"] + max(1, case["rows"] // 2)) // 2
        per = D * e if case["kind"] == "attend" else row4
        return {"bytes": C * H * (2 * slots * per + 2 * rows * G * D * e + (8 * slots if case["weights"] else 0)),
                "flops": 4 * D * pairs * C * H * G}
    n = C * case["layers"] * H
    if case["kind"] == "store4":
        return {"bytes": n * 2 * case["rows"] * 2 * (D * e + row4), "flops": 0}
    length = (case["least"] + case["tokens"]) // 2
    keep = min(length, case["budget"])
    return {"bytes": n * (4 * length + keep * (4 * D * e + 8)), "flops": 0}


# ---------------------------------------------------------------- in 64 bits
def _exact_attend(case, q, keys, values, lens, q_lens, weights):
    """Head by head: the visible logits, their softmax and the sums, f64."""
    C, n, Hq, D = q.shape
    T, G = case["tokens"], case["group"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    got = weights.double() if weights is not None else None
    j = torch.arange(T, device=q.device)
    step = max(1, (1 << 27) // T)
    for c in range(C):
        length = int(lens[c])
        m = n if q_lens is None else int(q_lens[c])
        for h in range(Hq):
            K, V = keys[c, h // G, :length].double(), values[c, h // G, :length].double()
            for a in range(0, m, step):
                z = min(m, a + step)
                p = length - m + torch.arange(a, z, device=q.device).unsqueeze(1)
                hide = j[:length].unsqueeze(0) > p
                if case["window"]:
                    hide |= (j[:length].unsqueeze(0) <= p - case["window"]) & (j[:length].unsqueeze(0) >= case["sinks"])
                t = (q[c, a:z, h].double() @ K.T) / math.sqrt(D)
                t[hide] = -math.inf
                t = torch.softmax(t, dim=1)
                t[hide.all(dim=1)] = 0.0
                out[c, a:z, h] = t @ V
                if got is not None:
                    got[c, h // G, :length] += t.sum(dim=0)
    return {"out": out} if got is None else {"out": out, "weights": got}


def _exact_values(codes, scales):
    """What the 4-bit codes stand for, by a table of all 16, f64."""
    table = torch.tensor(GRID + tuple(-g for g in GRID), dtype=torch.float64, device=codes.device)
    low, high = table[(codes % 16).long()], table[(codes // 16).long()]
    v = torch.stack((low, high), dim=-1).flatten(-2)
    return v * torch.pow(2.0, scales.double() - 127.0).repeat_interleave(BLOCK, dim=-1)


def _exact_store(x):
    """The nearest representable value of each element under its block's scale,
    f64: by distance to every grid value, ties to the even code."""
    b = x.double().reshape(*x.shape[:-1], -1, BLOCK)
    top = b.abs().amax(dim=-1)
    e = torch.ceil(torch.log2(top.clamp(min=1e-300) / 7.0))
    e = torch.where(7.0 * torch.pow(2.0, e - 1) >= top, e - 1, e)      # log2's last bit
    e = torch.where(7.0 * torch.pow(2.0, e) < top, e + 1, e).clamp(-125, 125)
    size = torch.pow(2.0, e).unsqueeze(-1)
    out = torch.zeros_like(b)
    best = torch.full_like(b, math.inf)
    a = b.abs() / size
    for code in (0, 2, 4, 6, 1, 3, 5, 7):                              # even codes first: they win ties
        d = (a - GRID[code]).abs()
        out = torch.where(d < best, torch.full_like(b, GRID[code]), out)
        best = torch.minimum(best, d)
    return (torch.copysign(out, b) * size).reshape(x.shape)


def _exact_evict(case, buf, weights, lens):
    """Head by head: the middle slots in order of (weight falling, slot rising),
    cut at the budget; rows and weights moved as they are."""
    C, L, H, _ = weights.shape
    B = case["budget"]
    out = torch.zeros((C, L, 2, H, B, case["dim"]), dtype=torch.float64, device=buf.device)
    kept = torch.full((C, L, H, B), -1, dtype=torch.int32)
    moved = torch.zeros((C, L, H, B), dtype=torch.float64)
    for c, n in enumerate(lens):
        first, last = min(case["sinks"], n), max(0, n - case["recent"])
        for layer in range(L):
            for h in range(H):
                slots = list(range(n))
                if n > B:
                    w = weights[c, layer, h].tolist()
                    middle = sorted(range(first, last), key=lambda j: (-w[j], j))
                    slots = sorted(slots[:first] + slots[last:] + middle[:B - first - (n - last)])
                at = torch.tensor(slots)
                kept[c, layer, h, :len(slots)] = at.to(torch.int32)
                moved[c, layer, h, :len(slots)] = weights[c, layer, h][at].double()
                out[c, layer, :, h, :len(slots)] = buf[c, layer, :, h][:, at.to(buf.device)].double()
    return {"buf": out, "weights": moved, "kept": kept, "lens": torch.tensor([min(n, B) for n in lens])}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attend":
        x = s["buf"][:, 0]
        return _exact_attend(case, s["q"], x[:, 0], x[:, 1], s["lens"], s["q_lens"], s["weights"])
    if case["kind"] == "attend4":
        x = _exact_values(s["codes"][:, 0], s["scales"][:, 0])
        return _exact_attend(case, s["q"], x[:, 0], x[:, 1], s["lens"], s["q_lens"], s["weights"])
    if case["kind"] == "store4":
        return {"keys": _exact_store(s["keys"]), "values": _exact_store(s["values"])}
    return _exact_evict(case, s["buf"], s["weights"].cpu(), s["lens"].tolist())
