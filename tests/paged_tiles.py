"""Calls that reach each tile of the many-row attention kernel (256, 128 and 64
rows), over pages and of packed prompts: their sizes, the rows a tile that the
library chooses for them and whether a join follows; and the plain form of
paged_ref.attend, a sequence at a time."""
import math

import torch

# name: rows a tile, joined, heads, group, rows of each sequence, their lengths, page, window, sinks
PAGED = {
    "256 short": (256, False, 32, 1, [130] * 5, [130, 260, 300, 131, 400], 16, 0, 0),
    "256 long": (256, True, 32, 1, [1100], [2000], 64, 0, 0),
    "256 window": (256, True, 32, 1, [1100, 3], [2000, 90], 32, 700, 4),
    "256 mixed": (256, True, 16, 2, [700, 1, 650, 40], [1500, 900, 650, 30], 16, 0, 0),
    "256 group": (256, True, 8, 4, [1000, 200], [2100, 200], 128, 0, 0),
    "128 join": (128, True, 32, 1, [300, 200], [1000, 700], 64, 0, 0),
    "128 window": (128, False, 32, 1, [300, 200], [1000, 700], 16, 300, 70),
    "128 long": (128, True, 16, 1, [1100, 1], [2000, 2000], 64, 0, 0),
    "64 join": (64, True, 4, 1, [300, 200], [3000, 900], 64, 0, 0),
    "64 tokens": (64, True, 8, 20, [1, 2, 1], [1500, 70, 1], 32, 0, 0),
}
# name: rows a tile, joined, heads, group, rows of each sequence, window, sinks
PROMPTS = {
    "256 short": (256, False, 32, 1, [130] * 5, 0, 0),
    "256": (256, False, 32, 1, [600, 0, 100, 40], 0, 0),
    "256 long": (256, True, 32, 1, [1500], 0, 0),
    "256 window": (256, True, 32, 1, [1500, 7], 800, 5),
    "256 group": (256, True, 8, 4, [1400, 300], 0, 0),
    "128": (128, False, 32, 1, [300, 200], 0, 0),
    "128 long": (128, True, 16, 1, [1500, 40], 0, 0),
    "128 window": (128, False, 32, 1, [300, 200], 150, 3),
    "64 long": (64, True, 8, 1, [1500], 0, 0),
}
SCALE = {64: 0.125, 128: 1 / math.sqrt(128)}


def table_pages(lens, page):
    return max((n + page - 1) // page for n in lens)


def small_weights(ref, dtype):
    """ref with room for weights that count as 0, where bf16 products' weighted
    sums pass the end of 32 bits.  A row's largest weight is then held as 2^-40 or
    more (up to 2^8 of the lag under it), and one below 2^-126, the smallest normal
    number, may be held as 0: each is off by at most 2^-126 / 2^-40 = 2^-86 of the
    largest, the row by at most 2^-86 sum |v|, since what it is divided by is no
    less than the largest.  out_bound takes half a step of the type times mass."""
    half = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    return dict(ref, mass=ref["mass"] + 2.0 ** -86 / half * ref["total"])


def attend(q, kv, lens, spans, window, sinks, scale):
    """paged_ref.attend's fields; where there is a GPU, 64-bit products on it."""
    rows, Hq, D = q.shape
    on = dict(dtype=torch.float64, device="cuda" if torch.cuda.is_available() else "cpu")
    q, out = q.to(**on), torch.zeros(rows, Hq, D, **on)
    mass, total = torch.zeros_like(out), torch.zeros_like(out)
    dev, count = torch.zeros(rows, Hq, **on), torch.zeros(rows, Hq, **on)
    lse = torch.full((Hq, rows), -math.inf, **on)
    for (K, V, there), n, (a, m) in zip(kv, lens, spans):
        if not m or not n:
            continue
        G, K, V, there = Hq // K.shape[0], K.to(**on), V.to(**on), there.to(on["device"])
        pos, j = torch.arange(n - m, n, device=on["device"])[:, None], torch.arange(n, device=on["device"])
        see = (j <= pos) & there[:n]
        if window:
            see &= (pos - j < window) | (j < sinks)
        some = see.any(1)
        V = torch.where(there[:n, None], V, 0.0)
        finite = torch.isfinite(V)
        odd = (~finite).nonzero().tolist()
        for h in range(K.shape[0]):
            v = torch.where(finite[h], V[h], 0.0)
            sums = see.double() @ v.abs()
            for g in range(h * G, h * G + G):
                x = q[a:a + m, g]
                s = torch.where(see, (x @ K[h].T) * scale, -math.inf)
                p = torch.where(some[:, None], torch.softmax(s, 1), 0.0)
                o, ma, to = p @ v, p @ v.abs(), sums.clone()
                for _, j, d in (z for z in odd if z[0] == h):
                    at = see[:, j]
                    o[at, d] += p[at, j] * V[h, j, d]
                    ma[at, d] += p[at, j] * V[h, j, d].abs()
                    to[at, d] += V[h, j, d].abs()
                out[a:a + m, g], mass[a:a + m, g], total[a:a + m, g] = o, ma, to
                lse[g, a:a + m] = torch.logsumexp(s, 1)
                big = torch.where(see, x.abs() @ K[h].abs().T, 0.0).amax(1)
                high = torch.where(see, s.abs(), 0.0).amax(1)
                d = (D + 4) * scale * big + 4 * high + 8
                dev[a:a + m, g] = torch.where(some, d, 0.0)
                count[a:a + m, g] = see.sum(1).double()
    return {name: x.cpu() for name, x in dict(out=out, lse=lse, mass=mass, total=total, dev=dev, count=count).items()}
