"""Plain 64-bit forms of the paged-cache operators on the CPU: what 8-bit pages
hold, and attention of packed rows, with what live_ref's error bounds go by."""
import math

import torch

import live_ref as R


def table8():
    """The 256 values of e4m3: 4 exponent bits of bias 7, 3 of mantissa, no infinity."""
    v = []
    for c in range(256):
        e, m = c >> 3 & 15, c & 7
        x = math.nan if c & 127 == 127 else m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        v.append(-x if c & 128 else x)
    return torch.tensor(v, dtype=torch.float64)


def values(buf, scales=None):
    """f64 values of pages, on the CPU."""
    if scales is None:
        return buf.cpu().double()
    s = scales.cpu().long()
    p = torch.where(s == 255, torch.tensor(math.nan, dtype=torch.float64), torch.pow(2.0, (s - 127).double()))
    return table8()[buf.cpu().view(torch.uint8).long()] * p.repeat_interleave(32, -1)


def round8(x):
    """f64 values that rows x [.., dim] stand for after a store into 8-bit pages."""
    b = x.cpu().double().reshape(*x.shape[:-1], -1, 32)
    top = b.abs().amax(-1)
    e = torch.full(top.shape, -116, dtype=torch.int64)
    for k in range(-116, 119):
        e = torch.where(top > 448.0 * 2.0 ** k, k + 1, e)
    step = torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double()).unsqueeze(-1)
    grid = table8()[:127]                              # 0 .. 448, ascending by code
    y = (b.abs() / step).clamp(max=448.0)
    hi = torch.searchsorted(grid, y.contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    dl, dh = y - grid[lo], grid[hi] - y
    pick = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    v = torch.copysign(grid[pick], b) * step
    bad = ~torch.isfinite(top)
    return torch.where(bad.unsqueeze(-1), torch.full_like(v, math.nan), v).reshape(x.shape)


def rounded(x, dtype):
    return round8(x) if dtype in (torch.uint8, torch.float8_e4m3fn) else x.cpu().to(dtype).double()


def rows_of(starts, seqs, rows):
    """[(first, count)] of the sequences."""
    if starts is None:
        return [(s * (rows // seqs), rows // seqs) for s in range(seqs)]
    return [(a, z - a) for a, z in zip(starts[:-1], starts[1:])]


def gathered(pages, table, length):
    """(K, V [heads, length, dim], there [length]) of one sequence from pages [pages, 2, heads, P, dim]."""
    n, P = pages.shape[0], pages.shape[3]
    slot = torch.arange(length)
    page = torch.tensor([int(table[j // P]) for j in range(length)], dtype=torch.long)
    there = (page >= 0) & (page < n)
    x = pages[torch.where(there, page, 0), :, :, slot % P]         # [length, 2, heads, dim]
    return x[:, 0].transpose(0, 1), x[:, 1].transpose(0, 1), there


def attend(q, kv, lens, spans, window, sinks, scale):
    """q [rows, Hq, D] f64; kv[s] = (K, V, there); spans[s] = (first row, count).
    Fields as live_ref.attend's, rows packed: out, mass, total [rows, Hq, D], dev,
    count [rows, Hq], lse [Hq, rows]."""
    rows, Hq, D = q.shape
    out = torch.zeros(rows, Hq, D, dtype=torch.float64)
    mass, total = torch.zeros_like(out), torch.zeros_like(out)
    dev, count = (torch.zeros(rows, Hq, dtype=torch.float64) for _ in range(2))
    lse = torch.full((Hq, rows), -math.inf, dtype=torch.float64)
    for (K, V, there), n, (a, m) in zip(kv, lens, spans):
        H = K.shape[0]
        G = Hq // H
        for i in range(m):
            pos = n - m + i
            if pos < 0:
                continue
            at = (R.seen(pos, n, window, sinks) & there[:n]).nonzero().flatten()
            if not len(at):
                continue
            k, v = K[:, at], V[:, at]                                  # [H, slots, D]
            x = q[a + i].view(H, G, D)
            s = (x @ k.transpose(1, 2)) * scale                        # [H, G, slots]
            some = ~(s == -math.inf).all(-1)
            p = torch.where(some[..., None], torch.softmax(s, -1), torch.zeros(()).double())
            out[a + i] = (p @ v).view(Hq, D)
            lse[:, a + i] = torch.logsumexp(s, -1).view(Hq)
            mass[a + i] = (p @ v.abs()).view(Hq, D)
            total[a + i] = v.abs().sum(1).repeat_interleave(G, 0)
            # D products and D sums in 32 bits, the scale, exp's argument and result
            big = (x.abs() @ k.abs().transpose(1, 2)).amax(-1)
            dev[a + i] = ((D + 4) * scale * big + 4 * s.abs().amax(-1) + 8).view(Hq)
            count[a + i] = len(at)
    return dict(out=out, lse=lse, mass=mass, total=total, dev=dev, count=count)


def lse_bound(ref):
    return R.lse_bound(dict(lse=ref["lse"][None], dev=ref["dev"][None], count=ref["count"][None]))[0]


def check(out, lse, ref, spans, dtype, before=None, lse_before=None):
    """Every row of a sequence within its bound, the others as they were."""
    o, mine = out.cpu().double(), torch.zeros(out.shape[0], dtype=torch.bool)
    for a, m in spans:
        mine[a:a + m] = True
    err = (o - ref["out"]).abs() - R.out_bound(ref, dtype)
    both = torch.isnan(o) & torch.isnan(ref["out"])
    err = torch.where(both | (o == ref["out"]), torch.full_like(err, -1.0), err)[mine]
    assert not torch.isnan(err).any() and not (err > 0).any(), f"out over its bound by {err.max()}"
    if before is not None:
        assert R.same(o[~mine], torch.full_like(o[~mine], before)), "rows of nobody were written"
    if lse is not None:
        a, b = lse.cpu().double(), ref["lse"]
        fin = torch.isfinite(b) & mine
        assert R.same(torch.isinf(a[:, mine]), torch.isinf(b[:, mine]))
        assert ((a - b).abs()[fin] <= lse_bound(ref)[fin]).all()
        if lse_before is not None:
            assert R.same(a[:, ~mine], torch.full_like(a[:, ~mine], lse_before))
