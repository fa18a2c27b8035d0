"""Plain 64-bit restatement of the paged context operators (one context, one page, one head at a time), for the tests."""
import math

import torch

WIDTHS = (16, 32, 64, 96, 128, 256)
U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def width(hd):
    return next(w for w in WIDTHS if w >= hd)


def make_pages(num_pages, heads, page, hd, dtype, seed=0, fill=None):
    """Pages with every slot written (``fill``: with that value), padding channels zero."""
    g = torch.Generator().manual_seed(seed)
    w = width(hd)
    keys = torch.zeros(num_pages, heads, page, w, dtype=dtype)
    values = torch.zeros(num_pages, heads, w, page, dtype=dtype)
    keys[..., :hd] = torch.randn(num_pages, heads, page, hd, generator=g).to(dtype) if fill is None else fill
    values[:, :, :hd] = (torch.randn(num_pages, heads, hd, page, generator=g) + 0.5).to(dtype) if fill is None else fill
    return keys, values, keys.amin(2).contiguous(), keys.amax(2).contiguous()


def make_table(need, slots, num_pages, seed=0):
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(num_pages, generator=g).tolist()
    table = torch.full((len(need), slots), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        for s in range(n):
            table[b, s] = order.pop()
    return table


def rotate(k, positions, rotary, heads, hd, base=10000.0):
    """k [n, heads * hd] in 64 bits."""
    k = k.double().clone()
    if positions is None:
        return k
    n, axes = positions.shape
    row = heads * hd
    rotary = row if rotary is None else rotary
    span = rotary // axes
    starts = [0] if rotary > hd else [h * hd for h in range(heads)]
    out = k.clone()
    for first in starts:
        for a in range(axes):
            for j in range(span // 2):
                c = first + a * span + 2 * j
                angle = positions[:, a].double() * base ** (-2.0 * j / span)
                out[:, c] = k[:, c] * angle.cos() - k[:, c + 1] * angle.sin()
                out[:, c + 1] = k[:, c + 1] * angle.cos() + k[:, c] * angle.sin()
    return out


def append(pages, k, v, offsets, starts, table, hd, positions=None, rotary=None, base=10000.0):
    """(keys, values) in 64 bits after the append, and the set of (page, slot) written."""
    keys, values = pages[0].double(), pages[1].double()
    heads, page = keys.shape[1], keys.shape[2]
    k64 = rotate(k, positions, rotary, heads, hd, base)
    written = []
    for b in range(len(starts)):
        for i in range(int(offsets[b]), int(offsets[b + 1])):
            place = int(starts[b]) + i - int(offsets[b])
            if place // page >= table.shape[1]:
                continue
            p = int(table[b, place // page])
            if not 0 <= p < keys.shape[0]:
                continue
            keys[p, :, place % page, :hd] = k64[i].view(heads, hd)
            values[p, :, :hd, place % page] = v[i].double().view(heads, hd)
            written.append((p, place % page))
    return keys, values, written


def context(pages, table_row, length, h, hd):
    """(k [n, hd], v [n, hd]) of a context's tokens that are there, and their places."""
    keys, values = pages[0], pages[1]
    page = keys.shape[2]
    k, v, places = [], [], []
    for place in range(min(length, table_row.numel() * page)):
        p = int(table_row[place // page])
        if 0 <= p < keys.shape[0]:
            k.append(keys[p, h, place % page, :hd])
            v.append(values[p, h, :hd, place % page])
            places.append(place)
    if not k:
        return torch.zeros(0, hd).double(), torch.zeros(0, hd).double(), torch.zeros(0, dtype=torch.long)
    return torch.stack(k).double(), torch.stack(v).double(), torch.tensor(places)


def attention(q, pages, table, lengths, heads, hd, scale=None, selected=None):
    """(out in 64 bits, bound on the error of a kernel that sums in 32 bits and rounds once) [B, T, heads * hd].

    The bound: a logit is off by at most hd + 4 roundings of sum |q_c k_c| scale (products, the sum, the scale, the difference to the
    maximum), twice for the difference of two, the weights by the same factor and two ulp of the exponential; sums over n weights by n
    roundings; the two-part 16-bit weights by 2^-16, and by half's smallest step (2^-31 of the largest weight) each; then half a step
    of the type."""
    B, T, _ = q.shape
    H, page, dtype = pages[0].shape[1], pages[0].shape[2], q.dtype
    G = heads // H
    scale = hd ** -0.5 if scale is None else scale
    out = torch.zeros(B, T, heads, hd, dtype=torch.float64)
    bound = torch.zeros_like(out)
    for b in range(B):
        for h in range(H):
            k, v, places = context(pages, table[b], int(lengths[b]), h, hd)
            for t in range(T):
                keep = torch.ones(len(places), dtype=torch.bool)
                if selected is not None:
                    keep = torch.isin(places // page, selected[b, t, h].long())
                kk, vv = k[keep], v[keep]
                if len(kk) == 0:
                    continue
                for g in range(G):
                    x = q[b, t].view(heads, hd)[h * G + g].double()
                    logits = kk @ x * scale
                    p = torch.softmax(logits, 0)
                    o = p @ vv
                    size = float((kk.abs() @ x.abs()).max()) * abs(scale)
                    parts = 0.0 if dtype == torch.float32 else 2.0 ** -16 + len(kk) * 2.0 ** -31
                    rel = 2 * (hd + 4) * U * size + (len(kk) + 8) * U + parts
                    out[b, t, h * G + g] = o
                    bound[b, t, h * G + g] = 2 * rel * (p @ vv.abs()) + HALF_STEP[dtype] * o.abs() * (1 + rel) + 2.0 ** -25 * (dtype == torch.float16)
    return out.view(B, T, -1), bound.view(B, T, -1)


def select(q, key_min, key_max, table, lengths, page, heads, hd, count):
    B, T, _ = q.shape
    H = key_min.shape[1]
    G = heads // H
    out = torch.full((B, T, H, count), -1, dtype=torch.int32)
    for b in range(B):
        slots = [s for s in range(table.shape[1]) if 0 <= int(table[b, s]) < key_min.shape[0] and s * page < int(lengths[b])]
        for t in range(T):
            for h in range(H):
                scored = []
                for s in slots:
                    lo, hi = key_min[int(table[b, s]), h, :hd].double(), key_max[int(table[b, s]), h, :hd].double()
                    best = -math.inf
                    for g in range(G):
                        x = q[b, t].view(heads, hd)[h * G + g].double()
                        best = max(best, float((x.clamp(min=0) * hi + x.clamp(max=0) * lo).sum()))
                    scored.append((-best, s))
                chosen = sorted(s for _, s in sorted(scored)[:count])
                out[b, t, h, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
    return out
