"""Plain 64-bit forms of the live-cache operators on the CPU, and the error
bounds that the tests of the kernels go by."""
import math

import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def same(a, b):
    """Equal values (NaN equals NaN), without a dump of both when they are not."""
    a, b = a.detach().cpu(), b.detach().cpu()
    return a.shape == b.shape and a.dtype == b.dtype and bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


def fp4_values(codes, scales):
    """f64 values of codes [.., dim / 2] and scale bytes [.., dim / 32]."""
    codes, scales = codes.cpu().long(), scales.cpu().long()
    c = torch.stack((codes % 16, codes // 16), -1).flatten(-2)
    v = GRID[c % 8] * torch.where(c >= 8, -1.0, 1.0)
    s = torch.where(scales == 255, torch.tensor(math.nan, dtype=torch.float64),
                    torch.pow(torch.tensor(2.0, dtype=torch.float64), (scales - 127).double()))
    return v * s.repeat_interleave(32, -1)


def fp4_round(x):
    """f64 values that rows x [.., dim] stand for after a store: scale the
    smallest 2^e (e in -125 .. 125) with max |x| <= 7 * 2^e, nearest value,
    ties to the even code; NaN blocks for non-finite ones."""
    b = x.cpu().double().reshape(*x.shape[:-1], -1, 32)
    top = b.abs().amax(-1)
    e = torch.full(top.shape, -125, dtype=torch.int64)
    for k in range(-125, 125):
        e = torch.where(top > 7.0 * 2.0 ** k, k + 1, e)
    step = torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double()).unsqueeze(-1)
    d = ((b.abs() / step).unsqueeze(-1) - GRID).abs()
    low = d.amin(-1, keepdim=True)
    near = d == low                                   # one or two codes
    even = near & (torch.arange(8) % 2 == 0)
    pick = torch.where(even.any(-1, keepdim=True), even, near).double().argmax(-1)
    v = torch.copysign(GRID[pick], b) * step
    bad = ~torch.isfinite(top)
    return torch.where(bad.unsqueeze(-1), torch.full_like(v, math.nan), v).reshape(x.shape)


def seen(pos, n, window, sinks):
    j = torch.arange(n)
    ok = j <= pos
    if window:
        ok &= (pos - j < window) | (j < sinks)
    return ok


def attend(q, k, v, lens, q_lens, window, sinks, scale):
    """q [C, n, Hq, D], k / v [C, H, T, D] f64.  Returns out, lse, weights, and
    for the bounds: mass [.., D] = sum w |v|, total [.., D] = sum |v|, dev =
    bound of one logit's error in units of 2^-24, count of visible slots."""
    C, n, Hq, D = q.shape
    H, T = k.shape[1], k.shape[2]
    G = Hq // H
    out = torch.zeros(C, n, Hq, D, dtype=torch.float64)
    mass, total = torch.zeros_like(out), torch.zeros_like(out)
    lse = torch.full((C, Hq, n), -math.inf, dtype=torch.float64)
    dev = torch.zeros(C, n, Hq, dtype=torch.float64)
    count = torch.zeros(C, n, Hq, dtype=torch.float64)
    weights = torch.zeros(C, H, T, dtype=torch.float64)
    wdev = torch.zeros(C, H, T, dtype=torch.float64)
    for c in range(C):
        for i in range(q_lens[c]):
            pos = lens[c] - q_lens[c] + i
            at = seen(pos, T, window, sinks).nonzero().flatten() if pos >= 0 else torch.zeros(0, dtype=torch.long)
            if not len(at):
                continue
            for h in range(Hq):
                K, V = k[c, h // G, at], v[c, h // G, at]
                s = (K @ q[c, i, h]) * scale
                if bool((s == -math.inf).all()):
                    continue
                p = torch.softmax(s, 0)
                out[c, i, h] = p @ V
                lse[c, h, i] = torch.logsumexp(s, 0)
                mass[c, i, h] = p @ V.abs()
                total[c, i, h] = V.abs().sum(0)
                # D products and D sums in 32 bits, the scale, exp's argument and result
                dev[c, i, h] = (D + 4) * scale * (K.abs() @ q[c, i, h].abs()).max() + 4 * s.abs().max() + 8
                count[c, i, h] = len(at)
                weights[c, h // G, at] += p
                wdev[c, h // G, at] += p * 2 * dev[c, i, h]
    return dict(out=out, lse=lse, weights=weights, mass=mass, total=total, dev=dev, count=count, wdev=wdev)


def out_bound(ref, dtype):
    """|kernel - exact| at most: the rounding of the output, of each weight to
    the matrix products' type (16-bit calls; f16 weights below 2^-14 by
    2^-25 of the largest, 1), a weight's error from its logit and the
    normaliser's, and the sums' in 32 bits."""
    h, u = HALF[dtype], 2.0 ** -24
    rel = 2 * ref["dev"] * u + 4 * (ref["count"] + 16) * u
    b = h * ref["out"].abs() + (rel.unsqueeze(-1) + (h if dtype != torch.float32 else 0.0)) * ref["mass"] * (1 + h)
    if dtype == torch.float16:
        b = b + 2.0 ** -24 * ref["total"] + 2.0 ** -24
    return b + 1e-37


def lse_bound(ref):
    u = 2.0 ** -24
    lse = torch.where(torch.isfinite(ref["lse"]), ref["lse"].abs(), torch.zeros(()).double())
    return ref["dev"].permute(0, 2, 1) * u + 2 * (ref["count"].permute(0, 2, 1) + 8) * u + 4 * lse * u


def weights_bound(ref, before, rows):
    """`rows`: rows x group added up."""
    u = 2.0 ** -24
    n = ref["count"].max()
    return (ref["wdev"] + (4 * (n + 16) + rows) * ref["weights"] + 2 * before.double().abs()) * u + 1e-37


def evict(w, n, budget, sinks, recent):
    """Kept slots of one head, ascending."""
    if n <= budget:
        return list(range(n))
    mid = list(range(sinks, n - recent))
    val = [float(x) for x in w[:n]]
    val = [-math.inf if math.isnan(x) else x for x in val]
    mid.sort(key=lambda j: (-val[j], j))
    return sorted(list(range(sinks)) + mid[:budget - sinks - recent] + list(range(n - recent, n)))
