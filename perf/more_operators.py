"""The operators of a paged KV cache, as cases that can be timed and compared:
packed rows of sequences of different lengths stored into pages and read back
(16 bits, or 8 bits with a scale per 32 values), attention of single tokens and
of prompt chunks over the pages that a block table names, and attention of
whole packed prompts on their own rows.

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
BLOCK = 32                 # values that share one scale in 8-bit pages


def listed():
    return [
        # one new token of each of 64 conversations written to the 8-bit pages of
        # one layer and read back: the smallest store
        dict(name="store8_token", kind="store", dtype="bf16", cache="f8", layers=1, seqs=64, heads=8, dim=128, page=16,
             tokens=2048, least=40, rows=1, mixed=False),
        # prompts of six conversations, all 24 layers of the 32-head, head_dim-64
        # shape as the pool rehydrates them (f32), into 8-bit pages and back
        dict(name="store8_prompts", kind="store", dtype="f32", cache="f8", layers=24, seqs=6, heads=32, dim=64, page=64,
             tokens=1024, least=65, rows=1024, mixed=True),
        # one new token of one short conversation: the call where latency is
        # everything
        dict(name="paged_short", kind="attend", dtype="bf16", cache="bf16", seqs=1, heads=32, group=1, dim=64, page=16,
             tokens=700, least=700, shared=0, rows=1, mixed=False, window=0, sinks=0),
        # one new token of each of 8 agents that share the pages of a 768-token
        # prefix and have a few of their own
        dict(name="paged_agents", kind="attend", dtype="f16", cache="f16", seqs=8, heads=32, group=1, dim=64, page=32,
             tokens=1024, least=790, shared=768, rows=1, mixed=False, window=0, sinks=0),
        # one new token of 24 conversations from short to long, four query heads
        # to a KV head
        dict(name="paged_long", kind="attend", dtype="bf16", cache="bf16", seqs=24, heads=8, group=4, dim=128, page=64,
             tokens=32768, least=700, shared=0, rows=1, mixed=False, window=0, sinks=0),
        # the same conversations held in 8 bits, small pages
        dict(name="paged8_long", kind="attend", dtype="bf16", cache="f8", seqs=24, heads=8, group=4, dim=128, page=16,
             tokens=32768, least=700, shared=0, rows=1, mixed=False, window=0, sinks=0),
        # a full batch of middling conversations in 8 bits, eight query heads to a
        # KV head, 16-bit floats of the other kind
        dict(name="paged8_batch", kind="attend", dtype="f16", cache="f8", seqs=97, heads=4, group=8, dim=128, page=32,
             tokens=3000, least=33, shared=0, rows=1, mixed=False, window=0, sinks=0),
        # chunks of prompts and single tokens in one batch
        dict(name="paged_mixed", kind="attend", dtype="bf16", cache="bf16", seqs=20, heads=8, group=4, dim=128, page=64,
             tokens=6000, least=600, shared=0, rows=512, mixed=True, window=0, sinks=0),
        # chunks over 8-bit pages with a window and first tokens that stay visible
        dict(name="paged8_chunk", kind="attend", dtype="f16", cache="f8", seqs=3, heads=8, group=3, dim=64, page=16,
             tokens=9000, least=2000, shared=0, rows=701, mixed=True, window=1024, sinks=4),
        # a handful of short prompts
        dict(name="prompts_short", kind="prompts", dtype="f16", seqs=5, heads=32, group=1, dim=64, tokens=130, least=17,
             window=0, sinks=0),
        # prompts from a few tokens to thousands, packed, with a window
        dict(name="prompts_ragged", kind="prompts", dtype="bf16", seqs=17, heads=8, group=4, dim=128, tokens=4099,
             least=9, window=1500, sinks=4),
        # long prompts: the largest call
        dict(name="prompts_long", kind="prompts", dtype="bf16", seqs=3, heads=8, group=4, dim=128, tokens=8192,
             least=3500, window=0, sinks=0),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["store", "attend", "attend", "attend", "prompts", "prompts"])
    dim, heads, page = rng.choice([64, 128]), rng.randint(1, 16), rng.choice([16, 32, 64, 128, 256])
    if kind == "store":
        cache, dtype = rng.choice(["f8", "f8", "bf16", "f16"]), rng.choice(["f32", "bf16", "f16"])
        seqs, layers, tokens = _log(rng, 1, 64), rng.randint(1, 8), _log(rng, 16, 8192)
        while seqs * layers * heads * tokens * dim > 1 << 26:
            tokens //= 2
        tokens, mixed = max(tokens, 3), rng.random() < 0.6
        return dict(kind=kind, dtype=dtype, cache=cache, layers=layers, seqs=seqs, heads=heads, dim=dim, page=page,
                    tokens=tokens, least=rng.randint(3, tokens), rows=tokens if mixed else rng.randint(1, 3),
                    mixed=mixed)
    dtype, group = rng.choice(["bf16", "f16"]), rng.randint(1, 8)
    window = rng.choice([0, 0, _log(rng, 1, 8192)])
    sinks = rng.choice([0, 1, 4, 17]) if window else 0
    if kind == "prompts":
        seqs, tokens = _log(rng, 1, 32), _log(rng, 2, 6000)
        # the largest listed call's work, and the rows of one sequence against each other held at once
        while seqs * heads * group * tokens * tokens > 1 << 31 or heads * group * tokens * tokens > 1 << 30:
            if seqs > 2:
                seqs -= 1
            else:
                tokens //= 2
        return dict(kind=kind, dtype=dtype, seqs=seqs, heads=heads, group=group, dim=dim, tokens=tokens,
                    least=rng.randint(1, tokens), window=window, sinks=sinks)
    cache = rng.choice([dtype, "f8"])
    form = rng.choice(["token", "token", "few", "chunk"])
    rows = 1 if form == "token" else rng.randint(2, 16) if form == "few" else _log(rng, 17, 1024)
    seqs, tokens = _log(rng, 1, 64), max(_log(rng, 16, 32768), rows)
    # the plain form holds every row against every slot, and each sequence's slots
    while seqs * heads * group * rows * tokens > 1 << 29 or seqs * heads * tokens * dim > 1 << 28:
        if seqs > 1:
            seqs -= 1
        elif tokens > 2 * rows:
            tokens //= 2
        else:
            group = max(1, group // 2)
            heads = max(1, heads - 1)
    least = rng.randint(max(1, tokens // 8), tokens)
    return dict(kind=kind, dtype=dtype, cache=cache, seqs=seqs, heads=heads, group=group, dim=dim, page=page,
                tokens=tokens, least=least, shared=least // page * page if rng.random() < 0.3 else 0, rows=rows,
                mixed=rows > 1 and rng.random() < 0.7, window=window, sinks=sinks)


# ---------------------------------------------------------------- shapes
def _spread(case):
    """Lengths of the sequences: from `least` to `tokens`, evenly over their
    logarithm, the first the longest."""
    lo, hi = case["least"], case["tokens"]
    return [min(hi, max(lo, round(lo * (hi / lo) ** (1.0 if i == 0 else i * 0.6180339887 % 1.0))))
            for i in range(case["seqs"])]


def _counts(case, lens):
    """Rows of each sequence: `rows` each, or (mixed) one for every other
    sequence and a quarter of `rows` up to all of them for the rest; no more than
    the sequence has, except where every sequence has as many."""
    if not case["mixed"]:
        return [case["rows"]] * len(lens)
    return [min(n, 1 if i % 2 else max(1, round(case["rows"] * (1.0 if i == 0 else 0.25 + 0.75 * (i * 0.7548776662 % 1.0)))))
            for i, n in enumerate(lens)]


def _starts(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def _gen(seed, device="cuda"):
    g = torch.Generator(device=device)
    g.manual_seed(int(seed))
    return g


def _words(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _keys(shape, heads_axis, g):
    """Gaussian rows with per-channel scales and a few large channels, f32."""
    x = torch.randn(shape, generator=g, device="cuda")
    side = [1] * len(shape)
    side[heads_axis], side[-1] = shape[heads_axis], shape[-1]
    scale = torch.exp(0.3 * torch.randn(side, generator=g, device="cuda"))
    outlier = torch.rand(side, generator=g, device="cuda") < 0.03
    return x * torch.where(outlier, scale * 3.0, scale)


def _tables(case, lens, g):
    """(tables, pages): the pages of each sequence in no order, the shared ones
    first; entries behind a sequence's last page repeat its first page."""
    P, shared = case["page"], case.get("shared", 0) // case["page"]
    need = [(n + P - 1) // P for n in lens]
    pages = shared + sum(max(0, n - shared) for n in need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").tolist()
    common, order = order[:shared], order[shared:]
    tables, at = [], 0
    for n in need:
        mine = common[:n] + order[at:at + max(0, n - shared)]
        at += max(0, n - shared)
        tables.append(mine + mine[:1] * (max(need) - n))
    return _words(tables), pages


def prepare(case, seed):
    g = _gen(seed)
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    H, D = case["heads"], case["dim"]
    lens = _spread(case)
    mix = torch.randperm(len(lens), generator=g, device="cuda").tolist()
    s = dict(case=dict(case), kind=kind)
    if kind == "prompts":
        lens = [lens[i] for i in mix]
        s["starts_host"] = _starts(lens)
        s["starts"], total = _words(s["starts_host"]), sum(lens)
        # one projection's output: query heads, then keys, then values of a row
        G = case["group"]
        x = torch.randn((total, H * G + 2 * H, D), generator=g, device="cuda")
        x[:, H * G:H * G + H] = _keys((total, H, D), 1, g)
        x = x.to(dt)
        s["q"], s["k"], s["v"] = x[:, :H * G], x[:, H * G:H * G + H], x[:, H * G + H:]
        s["max_rows"] = max(lens)
        return s
    counts = _counts(case, lens)
    lens, counts = [lens[i] for i in mix], [counts[i] for i in mix]
    s["lens"], s["lens_host"], s["counts"], total = _words(lens), lens, counts, sum(counts)
    s["starts_host"] = _starts(counts)
    s["starts"] = _words(s["starts_host"]) if case["mixed"] else None
    s["max_rows"], s["max_len"] = max(counts), max(lens)
    s["tables"], pages = _tables(case, lens, g)
    layers, P = case.get("layers", 1), case["page"]
    shape = (layers, pages, 2, H, P)
    if kind == "store":
        s["keys"] = _keys((layers, total, H, D), 2, g).to(dt)
        s["values"] = torch.randn((layers, total, H, D), generator=g, device="cuda").to(dt)
        s["scales"] = None
        if case["cache"] == "f8":
            s["buf"] = torch.zeros((*shape, D), dtype=torch.uint8, device="cuda")
            s["scales"] = torch.zeros((*shape, D // BLOCK), dtype=torch.uint8, device="cuda")
        else:
            s["buf"] = torch.zeros((*shape, D), dtype=DTYPES[case["cache"]], device="cuda")
    else:
        s["q"] = torch.randn((total, H * case["group"], D), generator=g, device="cuda").to(dt)
        x = torch.stack((_keys((layers, pages, H, P, D), 2, g),
                         torch.randn((layers, pages, H, P, D), generator=g, device="cuda")), dim=2)
        s["scales"] = None
        if case["cache"] == "f8":
            s["buf"], s["scales"] = _quantise(x)
        else:
            s["buf"] = x.to(DTYPES[case["cache"]])
        del x
    if own:
        from provekv_amd.paged import PagedKVCache
        s["pages"] = PagedKVCache.over(s["buf"], s["scales"])
    return s


# ---------------------------------------------------------------- plain forms
def _power(e):
    """2^e, f32, exactly (e: whole numbers of -126 .. 127)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantise(x):
    """8-bit codes (e4m3) and scale bytes of f32 rows [.., dim]: blocks of 32, the
    smallest scale 2^e (e in -116 .. 119) with max |x| <= 448 * 2^e; a value goes
    to the nearest code, half way to the even one, the largest to 448."""
    b = x.reshape(*x.shape[:-1], -1, BLOCK)
    m, e = torch.frexp(b.abs().amax(dim=-1))
    e = (e - 9 + (m > 0.875).to(e.dtype)).clamp(-116, 119)
    e = torch.where(m == 0, torch.full_like(e, -116), e)
    y = (b * _power(-e.unsqueeze(-1))).clamp(-448.0, 448.0)
    return y.reshape(x.shape).to(torch.float8_e4m3fn).view(torch.uint8), (e + 127).to(torch.uint8)


def _values(codes, scales):
    """The f32 values that codes and scale bytes stand for."""
    v = codes.view(torch.float8_e4m3fn).float().reshape(*codes.shape[:-1], -1, BLOCK)
    return (v * _power(scales.int().unsqueeze(-1) - 127)).reshape(codes.shape)


def _where(s):
    """(page, place) of every packed row's slot."""
    case = s["case"]
    S, total = len(s["counts"]), s["starts_host"][-1]
    if s["starts"] is None:
        n = case["rows"]
        seq = torch.arange(S, device="cuda").repeat_interleave(n)
        pos = s["lens"].long().repeat_interleave(n) - n + torch.arange(n, device="cuda").repeat(S)
    else:
        row = torch.arange(total, device="cuda")
        seq = (row.unsqueeze(1) >= s["starts"][1:].long().unsqueeze(0)).sum(dim=1)
        pos = s["lens"].long()[seq] - s["starts"].long()[seq + 1] + row
    return s["tables"].long()[seq, pos // case["page"]], pos % case["page"]


def _plain_store(s):
    page, place = _where(s)
    rows = torch.stack((s["keys"], s["values"]), dim=2).float()          # [layers, rows, 2, heads, dim]
    f8 = s["scales"] is not None
    if f8:
        new, scales = _quantise(rows)
    else:
        new = rows.to(s["buf"].dtype)
    s["buf"][:, page, :, :, place] = new.permute(1, 0, 2, 3, 4)
    got = s["buf"][:, page, :, :, place].permute(1, 0, 2, 3, 4)
    if f8:
        s["scales"][:, page, :, :, place] = scales.permute(1, 0, 2, 3, 4)
        got = _values(got.contiguous(), s["scales"][:, page, :, :, place].permute(1, 0, 2, 3, 4))
    got = got.to(s["keys"].dtype)
    return {"keys": got[:, :, 0].contiguous(), "values": got[:, :, 1].contiguous()}


def _softmax(logit, see):
    """Weights over the last axis; zeros where nothing is seen."""
    logit = logit.masked_fill(~see, -math.inf)
    top = logit.amax(dim=-1, keepdim=True)
    p = torch.exp(logit - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(dim=-1, keepdim=True)
    return p / torch.where(total == 0, torch.ones_like(total), total)


def _see(case, pos, slot):
    see = slot <= pos
    if case["window"]:
        see = see & ((pos - slot < case["window"]) | (slot < case["sinks"]))
    return see


def _plain_attend(s):
    case, q = s["case"], s["q"]
    S, n, T, P = len(s["counts"]), s["max_rows"], s["max_len"], case["page"]
    H, G, D = case["heads"], case["group"], case["dim"]
    buf = s["buf"][0] if s["scales"] is None else _values(s["buf"][0], s["scales"][0])
    most = (T + P - 1) // P
    kv = buf[s["tables"].long()[:, :most]].permute(0, 2, 3, 1, 4, 5).reshape(S, 2, H, most * P, D)[:, :, :, :T].float()
    row = torch.arange(n, device="cuda")
    if s["starts"] is None:
        first = torch.arange(S, device="cuda") * n
        count = torch.full_like(first, n)
    else:
        first = s["starts"].long()[:-1]
        count = s["starts"].long()[1:] - first
    real = row.view(1, n) < count.view(S, 1)
    at = torch.where(real, first.view(S, 1) + row.view(1, n), torch.zeros((), dtype=torch.long, device="cuda"))
    x = q[at].float().reshape(S, n, H, G, D).permute(0, 2, 1, 3, 4).reshape(S, H, n * G, D)
    logit = torch.matmul(x, kv[:, 0].transpose(-1, -2).contiguous()).view(S, H, n, G, T) * (1.0 / math.sqrt(D))
    pos = ((s["lens"].long() - count).view(S, 1) + row.view(1, n)).view(S, 1, n, 1, 1)
    see = _see(case, pos, torch.arange(T, device="cuda"))
    p = _softmax(logit, see)
    del logit
    o = torch.matmul(p.view(S, H, n * G, T), kv[:, 1].contiguous())
    o = o.view(S, H, n, G, D).permute(0, 2, 1, 3, 4).reshape(S, n, H * G, D)
    # the padded rows' places, in order, are the packed rows
    place = torch.where(real, at, torch.full_like(at, q.shape[0])).view(-1)
    out = torch.zeros((q.shape[0] + 1, H * G, D), dtype=torch.float32, device="cuda")
    out[place] = o.reshape(S * n, H * G, D)
    return {"out": out[:-1].to(q.dtype)}


def _plain_prompts(s):
    case, starts = s["case"], s["starts_host"]
    H, G, D = case["heads"], case["group"], case["dim"]
    outs = []
    for a, z in zip(starts[:-1], starts[1:]):
        n = z - a
        x = s["q"][a:z].float().reshape(n, H, G, D).permute(1, 0, 2, 3).reshape(H, n * G, D)
        k = s["k"][a:z].float().permute(1, 2, 0).contiguous()
        v = s["v"][a:z].float().permute(1, 0, 2).contiguous()
        slot = torch.arange(n, device="cuda")
        p = _softmax(torch.matmul(x, k).view(H, n, G, n) * (1.0 / math.sqrt(D)), _see(case, slot.view(n, 1, 1), slot))
        o = torch.matmul(p.view(H, n * G, n), v)
        outs.append(o.view(H, n, G, D).permute(1, 0, 2, 3).reshape(n, H * G, D))
    return {"out": torch.cat(outs).to(s["q"].dtype)}


def run(state):
    s, kind = state, state["kind"]
    if own:
        case = s["case"]
        if kind == "store":
            cache = s["pages"]
            cache.store(s["keys"], s["values"], s["tables"], s["lens"], starts=s["starts"])
            keys, values = cache.load(s["keys"].shape[1], s["tables"], s["lens"], starts=s["starts"],
                                      dtype=s["keys"].dtype)
            return {"keys": keys, "values": values}
        if kind == "attend":
            return {"out": s["pages"].attend(0, s["q"], s["tables"], s["lens"], starts=s["starts"],
                                             window=case["window"], sinks=case["sinks"], max_rows=s["max_rows"],
                                             max_len=s["max_len"])}
        from provekv_amd.paged import attend_prompts
        return {"out": attend_prompts(s["q"], s["k"], s["v"], s["starts"], window=case["window"], sinks=case["sinks"],
                                      max_rows=s["max_rows"])}
    if kind == "store":
        return _plain_store(s)
    return _plain_attend(s) if kind == "attend" else _plain_prompts(s)


# ---------------------------------------------------------------- work
def _pairs(case, length, rows):
    """(visible (row, slot) pairs, visible slots from the first on) of the last
    `rows` rows of a sequence."""
    w, k = case["window"], case["sinks"]
    pairs, low = 0, length
    for p in range(length - rows + 1, length + 1):     # slots up to and with the row's own
        if p <= 0:
            continue
        a = max(0, p - w) if w else 0
        pairs += p - a + min(k, a)
        low = min(low, a)
    return pairs, length - low + min(k, low)


def work(case):
    H, D, e = case["heads"], case["dim"], BYTES[case["dtype"]]
    lens = _spread(case)
    if case["kind"] == "prompts":
        G, total = case["group"], sum(lens)
        pairs = sum(_pairs(case, n, n)[0] for n in lens)
        return {"bytes": total * H * D * e * (2 * G + 2), "flops": 4 * D * pairs * H * G}
    counts = _counts(case, lens)
    slot = D + D / BLOCK if case["cache"] == "f8" else 2 * D      # bytes of one row of one side
    if case["kind"] == "store":
        rows = sum(min(n, m) for n, m in zip(counts, lens))
        return {"bytes": case["layers"] * H * rows * 2 * 2 * (D * e + slot), "flops": 0}
    G, pairs, slots = case["group"], 0, 0
    for i, (n, m) in enumerate(zip(lens, counts)):
        a, b = _pairs(case, n, m)
        pairs += a
        slots += b - (min(b, case["shared"]) if i else 0)          # shared pages are read once
    return {"bytes": H * (2 * slots * slot + 2 * sum(counts) * G * D * e), "flops": 4 * D * pairs * H * G}


# ---------------------------------------------------------------- in 64 bits
def _table8():
    """The 256 values of e4m3 (no infinity; 0x7f and 0xff are not numbers)."""
    out = []
    for c in range(256):
        e, m = c >> 3 & 15, c & 7
        v = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        out.append(math.nan if c & 127 == 127 else -v if c & 128 else v)
    return torch.tensor(out, dtype=torch.float64, device="cuda")


def _two_to(e):
    """2^e in f64 by its bits."""
    return (e.long() + 1023 << 52).view(torch.float64)


def _exact_values(codes, scales):
    return _table8()[codes.long()] * _two_to(scales.long() - 127).repeat_interleave(BLOCK, dim=-1)


def _exact_round(x, cache):
    """The value a page of this type holds for each element of x, f64."""
    if cache != "f8":
        return x.to(DTYPES[cache]).double()
    b = x.double().reshape(*x.shape[:-1], -1, BLOCK)
    top = b.abs().amax(dim=-1)
    e = torch.ceil(torch.log2(top.clamp(min=1e-300) / 448.0))
    e = torch.where(448.0 * _two_to(e - 1) >= top, e - 1, e)              # log2's last bit
    e = torch.where(448.0 * _two_to(e) < top, e + 1, e).clamp(-116, 119)
    size = _two_to(e).unsqueeze(-1)
    a = b.abs() / size
    step = torch.full_like(a, 2.0 ** -9)                                  # eight steps to a binade from 2^-6 on
    for k in range(-6, 9):
        step = torch.where(a >= 2.0 ** k, torch.full_like(a, 2.0 ** (k - 3)), step)
    return (torch.copysign(torch.round(a / step) * step, b) * size).clamp(-448.0 * size, 448.0 * size).reshape(x.shape)


def _exact_rows(case, q, K, V, first, G):
    """q [n, Hq, D] at positions first, first + 1, ..; K, V [H, T, D], f64."""
    n, Hq, D = q.shape
    H, T = K.shape[0], K.shape[1]
    out = torch.zeros((n, Hq, D), dtype=torch.float64, device="cuda")
    slot = torch.arange(T, device="cuda")
    step = max(1, (1 << 27) // max(1, T * Hq))
    for a in range(0, n, step):
        z = min(n, a + step)
        p = first + torch.arange(a, z, device="cuda").view(-1, 1)
        hide = slot > p
        if case["window"]:
            hide = hide | ((slot <= p - case["window"]) & (slot >= case["sinks"]))
        x = q[a:z].double().view(z - a, H, G, D).permute(1, 2, 0, 3).reshape(H, G * (z - a), D)
        t = torch.bmm(x, K.transpose(1, 2).contiguous()).view(H, G, z - a, T) / math.sqrt(D)
        t = t.masked_fill(hide, -math.inf)
        t = torch.softmax(t, dim=-1).masked_fill(hide.all(dim=1).view(-1, 1), 0.0)
        o = torch.bmm(t.view(H, G * (z - a), T), V)
        out[a:z] = o.view(H, G, z - a, D).permute(2, 0, 1, 3).reshape(z - a, Hq, D)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "prompts":
        starts, outs = s["starts_host"], []
        for a, z in zip(starts[:-1], starts[1:]):
            K, V = (s[x][a:z].double().transpose(0, 1).contiguous() for x in ("k", "v"))
            outs.append(_exact_rows(case, s["q"][a:z], K, V, 0, case["group"]))
        return {"out": torch.cat(outs)}
    if case["kind"] == "store":
        return {"keys": _exact_round(s["keys"], case["cache"]), "values": _exact_round(s["values"], case["cache"])}
    outs = []
    for i, (n, m, a) in enumerate(zip(s["lens_host"], s["counts"], s["starts_host"])):
        pages = s["tables"][i, :(n + case["page"] - 1) // case["page"]].long()
        x = s["buf"][0][pages]
        x = x.double() if s["scales"] is None else _exact_values(x, s["scales"][0][pages])
        K, V = (x[:, side].transpose(0, 1).reshape(case["heads"], -1, case["dim"])[:, :n].contiguous() for side in (0, 1))
        outs.append(_exact_rows(case, s["q"][a:a + m], K, V, n - m, case["group"]))
    return {"out": torch.cat(outs)}
