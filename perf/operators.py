"""Timed cases of the paged context memory (nvblox_mindmap_amd/diffuser_actor/paged_context.py): keys and values of growing contexts kept
in pages, the attention that reads them, and the attention over the pages that a cheap score selects.

A context is a sequence of tokens (map vertices, image patches, time steps).  Its keys and values lie in pages of ``page`` tokens:

  keys    [pages, kv_heads, page, width]     a token's channels side by side
  values  [pages, kv_heads, width, page]     a channel's tokens side by side
  key_min, key_max [pages, kv_heads, width]  smallest and largest stored key of the page, channel by channel
  table   [contexts, slots] int32            page of a context's tokens slot * page .. (slot + 1) * page - 1; outside [0, pages): none

with ``width`` the head size rounded up to one of WIDTHS (the channels behind head_dim are zero).

``run`` computes an operator from elementary torch operations, or calls the framework where ``own`` is true."""
import math

import numpy as np
import torch

own = False

WIDTHS = (16, 32, 64, 96, 128, 256)
BASE = 10000.0  # of the position rotation
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


# ---- cases ---------------------------------------------------------------------------------------------------------------------
def _append(name, dtype, batch, tokens, held, ragged, kv_heads, head_dim, page, axes, rotary):
    return {"name": name, "op": "append", "dtype": dtype, "batch": batch, "tokens": tokens, "held": held, "ragged": ragged, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "axes": axes, "rotary": rotary}


def _attend(name, dtype, batch, queries, longest, ragged, heads, kv_heads, head_dim, page):
    return {"name": name, "op": "attend", "dtype": dtype, "batch": batch, "queries": queries, "longest": longest, "ragged": ragged, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page}


def _select(name, dtype, batch, queries, longest, ragged, heads, kv_heads, head_dim, page, count):
    return dict(_attend(name, dtype, batch, queries, longest, ragged, heads, kv_heads, head_dim, page), op="select", count=count)


def listed():
    return [
        # one more map vertex for one robot's memory, the policy's 8 heads of 15 channels and its three-axis code: latency alone
        _append("append_one_vertex", "float32", 1, 1, 2047, False, 8, 15, 64, 3, 120),
        # a training batch's worth of contexts (image patches and map vertices of 32 robots) taken up at once
        _append("append_contexts", "float32", 32, 3080, 616, True, 8, 15, 64, 3, 120),
        # one step of 256 sequences, shared key-value heads, far positions
        _append("append_step", "bfloat16", 256, 1, 30000, True, 8, 128, 64, 1, 128),
        # prompts of 16 sequences taken up at once
        _append("append_prompts", "float16", 16, 16384, 100, True, 8, 64, 128, 1, 64),
        # a denoising step's two trajectory tokens (two grippers) over one observation's context
        _attend("attend_gripper_tokens", "float32", 1, 2, 3080, False, 8, 8, 15, 64),
        # one new token of each of 64 sequences of all lengths
        _attend("attend_step", "bfloat16", 64, 1, 8191, True, 32, 8, 128, 64),
        # one new token over a very long cache: the split over its length decides
        _attend("attend_long", "bfloat16", 1, 1, 1000003, False, 32, 8, 128, 128),
        # 16 trajectory tokens of 32 robots over maps of up to 20 011 vertices
        _attend("attend_trajectories", "float16", 32, 16, 20011, True, 12, 12, 64, 32),
        # the same two trajectory tokens over a larger map, 16 pages each
        _select("select_gripper_tokens", "float32", 1, 2, 12320, False, 8, 8, 15, 32, 16),
        # one new token of each of 16 long sequences, 64 of up to 2 048 pages for every key-value head
        _select("select_step", "bfloat16", 16, 1, 131072, True, 32, 8, 128, 64, 64),
        # one new token over 31 251 pages: scoring the pages is most of the work
        _select("select_long", "float16", 1, 1, 1000003, False, 16, 4, 64, 32, 128),
        # several tokens that each choose for themselves, small pages
        _select("select_tokens", "float32", 4, 7, 20011, True, 12, 12, 32, 16, 33),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("append", "attend", "select"))
    dtype = rng.choice(("float32", "float16", "bfloat16"))
    size = 4 if dtype == "float32" else 2
    head_dim = rng.choice((15, 16, 24, 32, 64, 80, 96, 128, rng.randint(8, 128), rng.randint(8, 256)))
    kv_heads = rng.choice((1, 2, 4, 8, 12, rng.randint(1, 16)))
    page, ragged = rng.choice((16, 32, 64, 128, 256)), rng.random() < 0.7
    row = kv_heads * head_dim
    if op == "append":
        batch = _log(rng, 1, 256)
        most = max(1, int(5e8 / (4 * row * size * batch)))  # bytes of one pass: below the largest listed case's
        tokens = _log(rng, 1, min(16384, most, 400000 // batch))
        axes = rng.choice((1, 2, 3))
        rotary = rng.choice((0, row - row % (2 * axes) if row % (2 * axes) == 0 else 0, head_dim - head_dim % (2 * axes), head_dim - head_dim % (2 * axes)))
        return _append("", dtype, batch, tokens, rng.choice((0, _log(rng, 1, 30000 if batch < 64 else 2000))), ragged, kv_heads, head_dim, page, axes, rotary)
    groups, queries = rng.choice((1, 1, 2, 4, 8, rng.randint(1, 9))), rng.choice((1, 1, 2, _log(rng, 1, 16)))
    batch = _log(rng, 1, 64)
    if op == "attend":
        longest = _log(rng, 1, min(1000003, max(1, int(min(2e9 / (2 * size), 2e10 / (4 * queries * groups)) / (row * batch)))))
        return _attend("", dtype, batch, queries, longest, ragged, groups * kv_heads, kv_heads, head_dim, page)
    batch = min(batch, 16)
    longest = _log(rng, 1, min(1000003, max(1, int(2e9 / (2 * row * size * batch)))))
    slots = -(-longest // page)
    count = _log(rng, 1, max(1, min(256, slots, int(2.5e8 / (2 * row * size * batch * page * queries)))))
    return _select("", dtype, batch, queries, longest, ragged, groups * kv_heads, kv_heads, head_dim, page, count)


def _spread(most, batch, ragged, floor=0):
    """Lengths of a batch: all alike, or spread evenly from the longest down to an eighth of it, with an empty context among eight or more."""
    n = [most - (7 * most * i // (8 * batch) + i % 3 if ragged else 0) for i in range(batch)]
    n = [max(floor, x) for x in n]
    if ragged and batch >= 8:
        n[batch // 2] = floor
    return n


def _width(head_dim):
    return next(w for w in WIDTHS if w >= head_dim)


def _starts_counts(case):
    """Tokens that each context holds, and tokens that it gets (one at least in a step of single tokens)."""
    batch, ragged = case["batch"], case["ragged"]
    return _spread(case["held"], batch, ragged), _spread(case["tokens"], batch, ragged, 1 if case["tokens"] == 1 else 0)


def work(case):
    size, heads, hd, page = (4 if case["dtype"] == "float32" else 2), case["kv_heads"], case["head_dim"], case["page"]
    row = heads * hd * size
    if case["op"] == "append":
        starts, counts = _starts_counts(case)
        n = sum(counts)
        touched = sum(-(-(s + c) // page) - s // page for s, c in zip(starts, counts) if c)
        opened = sum(1 for s, c in zip(starts, counts) if c and s % page)  # pages whose earlier summary is read
        rotated = case["rotary"] * (1 if case["rotary"] > hd else heads)
        return {"bytes": n * (4 * row + (4 * case["axes"] if case["rotary"] else 0)) + 2 * row * (touched + opened) + 4 * (touched + 2 * case["batch"] + 1),
                "flops": n * (3 * rotated + 2 * heads * hd)}
    lengths = _spread(case["longest"], case["batch"], case["ragged"])
    group, queries, batch = case["heads"] // heads, case["queries"], case["batch"]
    qo = 2 * batch * queries * case["heads"] * hd * size
    pages = [-(-n // page) for n in lengths]
    if case["op"] == "attend":
        return {"bytes": 2 * row * sum(lengths) + qo + 4 * (sum(pages) + batch), "flops": 4 * queries * group * heads * hd * sum(lengths)}
    count = case["count"]
    read = sum(min(n, min(p, queries * count) * page) for n, p in zip(lengths, pages))
    dots = sum(min(n, min(p, count) * page) for n, p in zip(lengths, pages)) * queries
    return {"bytes": 2 * row * (sum(pages) + read) + qo + 4 * (sum(pages) + batch + batch * queries * heads * count),
            "flops": (2 * sum(pages) * queries + 4 * dots) * group * heads * hd}


# ---- inputs --------------------------------------------------------------------------------------------------------------------
def _table(lengths, page, generator, device):
    """Every context's pages, taken in any order from a pool that has a few more than are needed."""
    need = [-(-n // page) for n in lengths]
    pool = sum(need) + 3
    order = torch.randperm(pool, generator=generator, device=device).to(torch.int32)
    slots = max(max(need), 1)
    n = torch.tensor(need, device=device)
    at = torch.arange(slots, device=device)[None, :]
    first = torch.cumsum(n, 0) - n
    table = torch.where(at < n[:, None], order[torch.clamp(first[:, None] + at, max=pool - 1)], torch.full((), -1, dtype=torch.int32, device=device))
    return table.contiguous(), pool


def _pages(pool, heads, page, head_dim, dtype, generator, device):
    """Pages as earlier appends left them: keys of neighbouring tokens lie near each other (a page has a middle of its own), values have
    a mean for each channel."""
    w = _width(head_dim)
    rand = lambda *shape: torch.randn(shape, generator=generator, device=device, dtype=torch.float32)  # noqa: E731
    keys = torch.zeros((pool, heads, page, w), dtype=dtype, device=device)
    values = torch.zeros((pool, heads, w, page), dtype=dtype, device=device)
    mean = rand(heads, head_dim, 1)
    step = max(1, int(2e8) // (heads * page * head_dim))
    for a in range(0, pool, step):
        n = min(step, pool - a)
        keys[a:a + n, ..., :head_dim] = (0.8 * rand(n, heads, 1, head_dim) + 0.6 * rand(n, heads, page, head_dim)).to(dtype)
        values[a:a + n, :, :head_dim] = (mean + 0.7 * rand(n, heads, head_dim, page)).to(dtype)
    return keys, values


def prepare(case, seed):
    device, dtype = torch.device("cuda", torch.cuda.current_device()), DTYPES[case["dtype"]]
    g = torch.Generator(device=device).manual_seed(seed)
    heads, hd, page, batch = case["kv_heads"], case["head_dim"], case["page"], case["batch"]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    rand = lambda *shape: torch.randn(shape, generator=g, device=device, dtype=torch.float32)  # noqa: E731
    if case["op"] == "append":
        starts, counts = _starts_counts(case)
        table, pool = _table([s + c for s, c in zip(starts, counts)], page, g, device)
        keys, values = _pages(pool, heads, page, hd, dtype, g, device)
        n = sum(counts)
        offsets = np.concatenate([[0], np.cumsum(counts)]).tolist()
        if case["axes"] == 1:  # the token's place in its sequence; a far one in a third of the sequences
            place = torch.cat([torch.arange(s, s + c, device=device) + (100000 if b % 3 == 1 else 0) for b, (s, c) in enumerate(zip(starts, counts))])
            positions = place.to(torch.float32)[:, None].contiguous()
        else:  # points of the normalised workspace, or patch coordinates
            positions = 2 * torch.rand((n, case["axes"]), generator=g, device=device, dtype=torch.float32) - 1
        # keys and values are the halves of one projection's rows, as a key-value projection gives them
        kv = rand(n, 2 * heads * hd).to(dtype)
        return {"case": case, "keys": keys, "values": values, "key_min": keys.amin(2).contiguous(), "key_max": keys.amax(2).contiguous(), "kv": kv,
                "table": table, "starts": i32(starts), "offsets": i32(offsets), "positions": positions}
    lengths = _spread(case["longest"], batch, case["ragged"])
    table, pool = _table(lengths, page, g, device)
    keys, values = _pages(pool, heads, page, hd, dtype, g, device)
    q = (2.0 * rand(batch, case["queries"], case["heads"] * hd)).to(dtype)
    state = {"case": case, "keys": keys, "values": values, "q": q, "table": table, "lengths": i32(lengths)}
    if case["op"] == "select":
        state["key_min"], state["key_max"] = keys.amin(2).contiguous(), keys.amax(2).contiguous()
    return state


# ---- plain forms ---------------------------------------------------------------------------------------------------------------
def _rotated(k, positions, axes, rotary, heads, hd):
    """Keys [n, heads * hd] in 32 bits with channel pairs (2 i, 2 i + 1) turned by their position's angle: ``rotary`` channels, the axes
    one behind the other, pair i of an axis at BASE ** (-2 i / (rotary / axes)); of the whole row if rotary is wider than a head, else
    the first channels of every head."""
    if rotary == 0:
        return k
    span = rotary // axes
    frequency = torch.pow(BASE, -torch.arange(0, span, 2, device=k.device, dtype=torch.float64) / span)
    angle = (positions.double()[:, :, None] * frequency).flatten(1)  # far positions: 64 bits
    cos, sin = angle.cos().float(), angle.sin().float()
    x = k if rotary > hd else k.view(-1, heads, hd)
    if rotary <= hd:
        cos, sin = cos[:, None], sin[:, None]
    even, odd = x[..., 0:rotary:2], x[..., 1:rotary:2]
    turned = torch.stack((even * cos - odd * sin, odd * cos + even * sin), -1).flatten(-2)
    return torch.cat((turned, x[..., rotary:]), -1).reshape(k.shape)


def _plain_append(s):
    c = s["case"]
    heads, hd, page, dtype = c["kv_heads"], c["head_dim"], c["page"], s["keys"].dtype
    n, row = s["kv"].shape[0], heads * hd
    k = _rotated(s["kv"][:, :row].float(), s["positions"], c["axes"], c["rotary"], heads, hd).to(dtype).view(n, heads, hd)
    v = s["kv"][:, row:].reshape(n, heads, hd)
    token = torch.arange(n, device=k.device, dtype=torch.int32)
    context = torch.searchsorted(s["offsets"], token, right=True) - 1
    place = s["starts"][context] + token - s["offsets"][context]
    at, slot = s["table"][context, torch.div(place, page, rounding_mode="floor")].long(), (place % page).long()
    s["keys"][at, :, slot, :hd] = k
    s["values"][at, :, :hd, slot] = v
    # a page's summary begins anew with its first token: that one lifts the smallest and lowers the largest out of the way first
    low, high = s["key_min"][..., :hd], s["key_max"][..., :hd]
    lift = torch.where(slot == 0, math.inf, -math.inf).to(dtype)[:, None, None].expand(n, heads, hd)
    low.index_reduce_(0, at, lift, "amax")
    high.index_reduce_(0, at, -lift, "amin")
    low.index_reduce_(0, at, k, "amin")
    high.index_reduce_(0, at, k, "amax")
    return {"keys": s["keys"], "values": s["values"], "key_min": s["key_min"], "key_max": s["key_max"]}


def _softmax_sum(q, k, v, ignore, scale):
    """q [..., r, hd], k [..., L, hd], v [..., hd, L], ignore [..., 1, L]: softmax over the tokens that are not ignored; zeros where all are."""
    logits = (torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale).masked_fill(ignore, -math.inf)
    top = logits.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(logits - top)
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v.transpose(-1, -2).contiguous()) / torch.where(total > 0, total, torch.ones_like(total))


def _plain_attend(s):
    c = s["case"]
    heads, hd, page, dtype = c["kv_heads"], c["head_dim"], c["page"], s["q"].dtype
    b, t = s["q"].shape[:2]
    group = c["heads"] // heads
    at = s["table"].clamp(min=0).long()  # [b, slots]
    k = s["keys"][at][..., :hd].permute(0, 2, 1, 3, 4).reshape(b, heads, -1, hd).float()
    v = s["values"][at][..., :hd, :].permute(0, 2, 3, 1, 4).reshape(b, heads, hd, -1).float()
    q = s["q"].float().view(b, t, heads, group, hd).permute(0, 2, 1, 3, 4).reshape(b, heads, t * group, hd)
    ignore = (torch.arange(k.shape[2], device=k.device)[None, :] >= s["lengths"][:, None])[:, None, None, :]
    out = _softmax_sum(q, k, v.masked_fill(ignore, 0.0), ignore, 1.0 / math.sqrt(hd))
    return out.view(b, heads, t, group, hd).permute(0, 2, 1, 3, 4).reshape(b, t, -1).to(dtype)


def _plain_select(s):
    """Pages of every query token and key-value head: the bound that a page's smallest and largest keys put on the product of the query with
    any key in it, the largest over the heads that share the key-value head; the ``count`` best, the lower page first among equals."""
    c = s["case"]
    heads, hd, page, count = c["kv_heads"], c["head_dim"], c["page"], c["count"]
    b, t = s["q"].shape[:2]
    group, slots = c["heads"] // heads, s["table"].shape[1]
    at = s["table"].clamp(min=0).long()
    low = s["key_min"][at][..., :hd].permute(0, 2, 3, 1).double()  # [b, heads, hd, slots]; in 64 bits: the choice is a border
    high = s["key_max"][at][..., :hd].permute(0, 2, 3, 1).double()
    q = s["q"].double().view(b, t, heads, group, hd).permute(0, 2, 1, 3, 4).reshape(b, heads, t * group, hd)
    score = torch.matmul(q.clamp(min=0), high.contiguous()) + torch.matmul(q.clamp(max=0), low.contiguous())
    score = score.view(b, heads, t, group, slots).amax(3)
    there = (torch.arange(slots, device=q.device)[None, :] * page < s["lengths"][:, None])[:, None, None, :]
    score = score.masked_fill(~there, -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True)
    keep = min(count, slots)
    page_index = torch.where(order.values[..., :keep] > -math.inf, order.indices[..., :keep], slots).sort(-1).values
    chosen = torch.full((b, heads, t, count), -1, dtype=torch.int32, device=q.device)
    chosen[..., :keep] = torch.where(page_index < slots, page_index, -1).to(torch.int32)
    chosen = chosen.permute(0, 2, 1, 3).contiguous()  # [b, t, heads, count]

    pages = torch.gather(at[:, None, None, :].expand(b, t, heads, slots), 3, chosen.clamp(min=0).long())
    head = torch.arange(heads, device=q.device)[None, None, :, None]
    k = s["keys"][pages, head][..., :hd].reshape(b, t, heads, -1, hd).float()
    v = s["values"][pages, head][..., :hd, :].permute(0, 1, 2, 4, 3, 5).reshape(b, t, heads, hd, -1).float()
    place = chosen[..., None] * page + torch.arange(page, device=q.device)
    ignore = ((chosen[..., None] < 0) | (place >= s["lengths"][:, None, None, None, None])).reshape(b, t, heads, 1, -1)
    out = _softmax_sum(s["q"].float().view(b, t, heads, group, hd), k, v.masked_fill(ignore, 0.0), ignore, 1.0 / math.sqrt(hd))
    return {"pages": chosen, "out": out.reshape(b, t, -1).to(s["q"].dtype)}


# ---- the framework's calls -------------------------------------------------------------------------------------------------------
def _own(s):
    from nvblox_mindmap_amd.diffuser_actor import paged_context as P

    c = s["case"]
    pages = P.ContextPages(s["keys"], s["values"], s.get("key_min"), s.get("key_max"), c["head_dim"])
    if c["op"] == "append":
        row = c["kv_heads"] * c["head_dim"]
        P.append_context(pages, s["kv"][:, :row], s["kv"][:, row:], s["offsets"], s["starts"], s["table"],
                         s["positions"] if c["rotary"] else None, c["rotary"] or None)
        return {"keys": s["keys"], "values": s["values"], "key_min": s["key_min"], "key_max": s["key_max"]}
    if c["op"] == "attend":
        return P.context_attention(s["q"], pages, s["table"], s["lengths"], c["heads"])
    chosen = P.select_pages(s["q"], pages, s["table"], s["lengths"], c["heads"], c["count"])
    return {"pages": chosen, "out": P.context_attention(s["q"], pages, s["table"], s["lengths"], c["heads"], pages=chosen)}


def run(state):
    if own:
        return _own(state)
    return {"append": _plain_append, "attend": _plain_attend, "select": _plain_select}[state["case"]["op"]](state)


# ---- from the definitions, in 64 bits ----------------------------------------------------------------------------------------------
def _exact_append(s, starts, counts):
    c = s["case"]
    heads, hd, page, axes, rotary = c["kv_heads"], c["head_dim"], c["page"], c["axes"], c["rotary"]
    row = heads * hd
    kv = s["kv"].double()
    k, v = kv[:, :row].clone(), kv[:, row:]
    period = row if rotary > hd else hd
    if rotary:
        span = rotary // axes
        channel = torch.arange(row, device=k.device)
        within = channel % period
        pair = torch.div(within % span, 2, rounding_mode="floor").double()
        angle = s["positions"].double()[:, torch.div(within, span, rounding_mode="floor").clamp(max=axes - 1)] * torch.exp(-math.log(BASE) * 2 * pair / span)
        partner = torch.where(within % 2 == 0, channel + 1, channel - 1).clamp(0, row - 1)
        sign = torch.where(within % 2 == 0, -1.0, 1.0).double()
        k = torch.where(within < rotary, k * angle.cos() + sign * k[:, partner] * angle.sin(), k)
    out = {n: s[n].double() for n in ("keys", "values", "key_min", "key_max")}
    table, at = s["table"].cpu().tolist(), 0
    for b, (start, count) in enumerate(zip(starts, counts)):
        done = 0
        while done < count:
            place = start + done
            first, n, p = place % page, min(page - place % page, count - done), table[b][place // page]
            new_k = k[at:at + n].view(n, heads, hd).transpose(0, 1)
            out["keys"][p, :, first:first + n, :hd] = new_k
            out["values"][p, :, :hd, first:first + n] = v[at:at + n].view(n, heads, hd).permute(1, 2, 0)
            low, high = new_k.amin(1), new_k.amax(1)
            if first:
                low, high = torch.minimum(low, out["key_min"][p, :, :hd]), torch.maximum(high, out["key_max"][p, :, :hd])
            out["key_min"][p, :, :hd], out["key_max"][p, :, :hd] = low, high
            done, at = done + n, at + n
    return out


def _exact_rows(q, k, v):
    """q [r, hd], k [n, hd], v [hd, n] in 64 bits."""
    if k.shape[0] == 0:
        return torch.zeros_like(q)
    logits = (k @ q.T) / math.sqrt(q.shape[1])  # [n, r]
    return (v @ torch.exp(logits - torch.logsumexp(logits, 0))).T


def _exact_attend(s, lengths):
    c = s["case"]
    heads, hd, page = c["kv_heads"], c["head_dim"], c["page"]
    b, t = s["q"].shape[:2]
    group = c["heads"] // heads
    q, out = s["q"].double().view(b, t, heads, group, hd), torch.zeros((b, t, heads, group, hd), dtype=torch.float64, device=s["q"].device)
    for i, n in enumerate(lengths):
        pages = s["table"][i, :-(-n // page)].long()
        for h in range(heads):
            k = s["keys"][pages, h].double().reshape(-1, s["keys"].shape[-1])[:n, :hd]
            v = s["values"][pages, h].double().permute(1, 0, 2).reshape(s["keys"].shape[-1], -1)[:hd, :n]
            out[i, :, h] = _exact_rows(q[i, :, h].reshape(-1, hd), k, v).view(t, group, hd)
    return out.view(b, t, -1)


def _exact_select(s, lengths):
    c = s["case"]
    heads, hd, page, count = c["kv_heads"], c["head_dim"], c["page"], c["count"]
    b, t = s["q"].shape[:2]
    group = c["heads"] // heads
    q, out = s["q"].double().view(b, t, heads, group, hd), torch.zeros((b, t, heads, group, hd), dtype=torch.float64, device=s["q"].device)
    chosen = np.full((b, t, heads, count), -1, dtype=np.int32)
    for i, n in enumerate(lengths):
        pages = s["table"][i, :-(-n // page)].long()
        for h in range(heads):
            if n == 0:
                continue
            low, high = s["key_min"][pages, h, :hd].double(), s["key_max"][pages, h, :hd].double()
            for x in range(t):
                bound = torch.stack([torch.where(u >= 0, high, low) @ u for u in q[i, x, h]]).amax(0).cpu().numpy()
                best = np.sort(np.lexsort((np.arange(len(bound)), -bound))[:count])
                chosen[i, x, h, :len(best)] = best
                places = torch.from_numpy((best[:, None] * page + np.arange(page)).reshape(-1)).to(q.device)
                at = pages[torch.from_numpy(best).to(q.device)]
                k = s["keys"][at, h].double().reshape(-1, s["keys"].shape[-1])[places < n, :hd]
                v = s["values"][at, h].double().permute(1, 0, 2).reshape(s["keys"].shape[-1], -1)[:hd, places < n]
                out[i, x, h] = _exact_rows(q[i, x, h], k, v)
    return {"pages": torch.from_numpy(chosen), "out": out.view(b, t, -1)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s, *_starts_counts(case))
    lengths = _spread(case["longest"], case["batch"], case["ragged"])
    return _exact_attend(s, lengths) if case["op"] == "attend" else _exact_select(s, lengths)
