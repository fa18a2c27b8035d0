"""The paged context operators (diffuser_actor/paged_context.py, csrc/mmf_kernels_paged.hip) against a 64-bit restatement."""
import math

import pytest
import torch

import paged_reference as R
from nvblox_mindmap_amd.diffuser_actor import paged_context as P

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def dev_pages(pages, hd):
    return P.ContextPages(*(t.cuda() for t in pages), hd)


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


# ---- append ----------------------------------------------------------------------------------------------------------------------
APPEND = [
    # heads, head_dim, page, starts, counts, axes, rotary (None: none, "row", or channels of a head)
    (8, 15, 64, [2047], [1], 3, "row"),
    (8, 15, 64, [0, 5, 63, 64], [130, 0, 1, 77], 3, "row"),
    (8, 15, 16, [3, 0], [40, 16], 2, 12),
    (1, 16, 32, [31, 0, 7], [2, 33, 1], 1, 16),
    (3, 64, 16, [0, 9], [100, 7], 1, 64),
    (2, 128, 128, [120, 300], [20, 5], 1, 96),
    (2, 80, 256, [250, 0], [270, 3], 2, 80),
    (5, 7, 16, [1, 2, 3], [1, 1, 1], 3, 6),
    (2, 250, 16, [5], [23], 1, 250),
    (4, 24, 32, [0, 0, 0], [0, 0, 0], 3, "row"),
    (12, 32, 64, list(range(70)), [(7 * i) % 5 for i in range(70)], 4, 32),
    (4, 33, 32, [30], [40], 1, None),
    (8, 131, 16, [3], [21], 1, None),
    (8, 255, 32, [0, 40], [33, 9], 1, 254),
    (16, 64, 128, [7], [300], 1, "row"),
    (8, 20, 64, [0], [129], 2, 16),
    (6, 128, 256, [0, 200], [500, 100], 3, "row"),
]


def check_append(case, dtype, in_dtype, strided, seed=3):
    heads, hd, page, starts, counts, axes, rotary = case
    row, n = heads * hd, sum(counts)
    need = [-(-(s + c) // page) for s, c in zip(starts, counts)]
    pages = R.make_pages(sum(need) + 4, heads, page, hd, dtype, seed)
    table = R.make_table(need, max(need) + 1, sum(need) + 4, seed)
    g = torch.Generator().manual_seed(seed)
    behind = 3  # rows behind the last context's
    kv = torch.randn(n + behind, 2 * row + (1 if strided else 0), generator=g).to(in_dtype)
    k, v = (kv[:, :row], kv[:, row:2 * row]) if strided else (kv[:, :row].contiguous(), kv[:, row:].contiguous())
    positions = None
    if rotary is not None:
        positions = (torch.rand(n + behind, axes, generator=g) * 4 - 2)
        positions[::3] = torch.round(positions[::3] * 300000)  # far ones
    rotary = row if rotary == "row" else rotary
    offsets = i32([0] + torch.tensor(counts).cumsum(0).tolist())
    dev = dev_pages(pages, hd)
    kv_dev = kv.cuda()
    kd, vd = (kv_dev[:, :row], kv_dev[:, row:2 * row]) if strided else (k.cuda(), v.cuda())
    P.append_context(dev, kd, vd, offsets.cuda(), i32(starts).cuda(), table.cuda(), None if positions is None else positions.cuda(), rotary)
    torch.cuda.synchronize()
    keys, values, written = R.append(pages, k, v, offsets, starts, table, hd, positions, rotary)
    got_k, got_v = dev.keys.cpu(), dev.values.cpu()
    assert torch.equal(got_v, values.to(dtype)), "values"
    # a rotated key: two products, a sum and the rounding of cos / sin (2 ulp) and of the reduced angle (pi 2^-24): 12 U of |e| + |o|
    slack = 12 * R.U * 2 * float(k.abs().max() if k.numel() else 0)
    assert bool(((got_k.double() - keys).abs() <= R.HALF_STEP[dtype] * keys.abs() + slack + 2.0 ** -25 * (dtype == torch.float16)).all()), "keys"
    mask = torch.ones(got_k.shape[0], page, dtype=torch.bool)
    for p, s in written:
        mask[p, s] = False
    untouched = mask[:, None, :, None].expand_as(got_k)
    assert torch.equal(got_k[untouched], pages[0][untouched]), "slots that get no token stay as they were"
    # summaries: of the stored keys, begun anew by the first slot, else joined with what was there; untouched pages' stay
    low, high = pages[2].clone(), pages[3].clone()
    by_page = {}
    for p, s in written:
        by_page.setdefault(p, []).append(s)
    for p, slots in by_page.items():
        lo, hi = got_k[p][:, slots].amin(1), got_k[p][:, slots].amax(1)
        low[p, :, :hd] = (lo if 0 in slots else torch.minimum(lo, low[p]))[:, :hd]
        high[p, :, :hd] = (hi if 0 in slots else torch.maximum(hi, high[p]))[:, :hd]
    assert torch.equal(dev.key_min.cpu(), low) and torch.equal(dev.key_max.cpu(), high), "summaries"


@pytest.mark.parametrize("case", APPEND, ids=[f"{c[0]}x{c[1]}p{c[2]}r{c[6]}" for c in APPEND])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("strided", [False, True])
def test_append(case, dtype, strided):
    check_append(case, dtype, dtype, strided)
    if dtype != torch.float32:
        check_append(case, dtype, torch.float32, strided)


def test_append_drops_tokens_without_a_page():
    """Tokens behind the table or on an entry outside the pool are not stored; nothing else is touched."""
    pages = R.make_pages(6, 2, 16, 16, torch.float32)
    table = i32([[2, -1, 9, 5], [6, 0, -2, 1]])
    k, v = torch.randn(100, 32), torch.randn(100, 32)
    offsets, starts = i32([0, 80, 100]), i32([0, 50])
    dev = dev_pages(pages, 16)
    P.append_context(dev, k.cuda(), v.cuda(), offsets.cuda(), starts.cuda(), table.cuda())
    keys, values, _ = R.append(pages, k, v, offsets, starts, table, 16)
    assert torch.equal(dev.keys.cpu(), keys.float()) and torch.equal(dev.values.cpu(), values.float())
    # offsets and starts that make no sense store nothing out of place
    for off, st in (([0, 300, -5], [0, 0]), ([-7, 10, 20], [-3, 0]), ([0, 10, 20], [2 ** 31 - 1, 2 ** 30])):
        P.append_context(dev, k.cuda(), v.cuda(), i32(off).cuda(), i32(st).cuda(), i32([[-1] * 4] * 2).cuda())
    torch.cuda.synchronize()
    assert torch.equal(dev.keys.cpu(), keys.float()) and torch.equal(dev.values.cpu(), values.float())


def test_append_shows_a_nan_key_in_the_summary():
    pages = R.make_pages(2, 1, 16, 16, torch.float32)
    dev = dev_pages(pages, 16)
    k = torch.randn(20, 16)
    k[3, 5] = math.nan
    P.append_context(dev, k.cuda(), k.cuda(), i32([0, 20]).cuda(), i32([0]).cuda(), i32([[1, 0]]).cuda())
    assert torch.isnan(dev.key_min[1, 0]).nonzero().flatten().tolist() == [5] and torch.isnan(dev.key_max[1, 0]).nonzero().flatten().tolist() == [5]
    assert not torch.isnan(dev.key_min[0]).any()


def test_append_rotates_as_the_policy_does():
    """rotary over the whole row with three axes = layers.apply_rotary(k, *rotary3d(xyz)) (whose angles are 32-bit products)."""
    from nvblox_mindmap_amd.diffuser_actor.layers import apply_rotary, rotary3d

    xyz = (torch.rand(1, 200, 3) * 2 - 1).cuda()
    k = torch.randn(1, 200, 120).cuda()
    context = P.allocate_pages(8, 8, 15, 32)
    P.append_context(context, k[0], k[0], i32([0, 200]).cuda(), i32([0]).cuda(), torch.arange(8, dtype=torch.int32).cuda()[None].contiguous(), xyz[0].contiguous())
    got = context.keys[:7, :, :, :15].permute(0, 2, 1, 3).reshape(-1, 120)[:200]
    want = apply_rotary(k, *rotary3d(xyz, 120))[0]
    assert float((got - want).abs().max()) <= 16 * R.U * 2 * float(k.abs().max())


# ---- attention -----------------------------------------------------------------------------------------------------------------------
ATTEND = [
    # heads, kv_heads, head_dim, page, T, lengths
    (8, 8, 15, 64, 2, [1, 0, 63, 65, 257]),
    (8, 2, 16, 16, 1, [1, 2, 17, 31, 33, 0]),
    (6, 3, 24, 32, 3, [100, 5]),
    (4, 1, 64, 64, 1, [129, 64, 1]),
    (8, 1, 64, 16, 5, [300]),
    (3, 3, 80, 128, 2, [131, 127]),
    (18, 2, 96, 32, 1, [70]),
    (8, 2, 128, 256, 1, [513, 3]),
    (17, 1, 128, 64, 3, [90, 0]),
    (2, 1, 250, 16, 9, [49]),
    (2, 2, 256, 64, 1, [700]),
    (4, 4, 32, 16, 33, [40]),
]


def check_attention(case, dtype, seed=1, scale=None, selected_count=None, poison=False):
    heads, kv, hd, page, T, lengths = case
    need = [-(-n // page) for n in lengths]
    pool, slots = sum(need) + 2, max(need) + 1
    pages = R.make_pages(pool, kv, page, hd, dtype, seed)
    table = R.make_table(need, slots, pool, seed)
    g = torch.Generator().manual_seed(seed)
    q = (1.5 * torch.randn(len(lengths), T, heads * hd, generator=g)).to(dtype)
    selected = None
    if selected_count is not None:
        selected = torch.full((len(lengths), T, kv, selected_count), -1, dtype=torch.int32)
        for b in range(len(lengths)):
            for t in range(T):
                for h in range(kv):
                    choice = torch.randperm(slots, generator=g)[:selected_count]
                    keep = torch.rand(len(choice), generator=g) < 0.8
                    selected[b, t, h, :len(choice)] = torch.where(keep, choice, -1).to(torch.int32)
    dev = list(pages)
    if poison:  # what lies behind a context's length, and in pages that no context has, is anything
        dev = [t.clone() for t in pages[:2]]
        used = torch.zeros(pool, page, dtype=torch.bool)
        for b, n in enumerate(lengths):
            for place in range(n):
                used[int(table[b, place // page]), place % page] = True
        dev[0][~used[:, None, :, None].expand_as(dev[0])] = math.nan
        dev[1][~used[:, None, None, :].expand_as(dev[1])] = math.inf
        dev += [pages[2], pages[3]]
    got = P.context_attention(q.cuda(), dev_pages(dev, hd), table.cuda(), i32(lengths).cuda(), heads, scale, None if selected is None else selected.cuda())
    torch.cuda.synchronize()
    want, bound = R.attention(q, pages, table, lengths, heads, hd, scale, selected)
    assert got.dtype == dtype and bool(torch.isfinite(got).all())
    off = (got.cpu().double() - want).abs()
    assert bool((off <= bound).all()), (float(off.max()), float((off / bound.clamp(min=1e-30)).max()))


@pytest.mark.parametrize("case", ATTEND, ids=[f"{c[0]}/{c[1]}x{c[2]}p{c[3]}t{c[4]}" for c in ATTEND])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_attention(case, dtype):
    check_attention(case, dtype)
    check_attention(case, dtype, seed=2, scale=0.3, poison=True)


@pytest.mark.parametrize("case", ATTEND, ids=[f"{c[0]}/{c[1]}x{c[2]}p{c[3]}t{c[4]}" for c in ATTEND])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("count", [1, 3])
def test_attention_over_selected_pages(case, dtype, count):
    check_attention(case, dtype, seed=count, selected_count=count, poison=True)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("page", [16, 256])
def test_attention_split_over_a_long_context(dtype, page):
    """Long enough for many splits and (page 16) several windows of page entries; lengths that end inside a tile, a split, a page."""
    check_attention((4, 2, 32, page, 2, [4999, 1, 0, 2048]), dtype, seed=5)
    check_attention((2, 1, 16, page, 1, [20001]), dtype, seed=6, poison=True)


@pytest.mark.parametrize("hd", [15, 24, 64, 80, 128, 200])
@pytest.mark.parametrize("splits", [5, 20, 33, 47, 63, 64, 71])
def test_attention_joins_any_number_of_splits(hd, splits):
    """One context and one head: 256 keys a split, the last one short.  (The join's lanes each hold one split's weight.)"""
    n = 256 * splits - 37
    pages = R.make_pages(-(-n // 256), 1, 256, hd, torch.float16, splits)
    table = torch.arange(pages[0].shape[0], dtype=torch.int32)[None].contiguous()
    q = (2 * torch.randn(1, 1, hd, generator=torch.Generator().manual_seed(splits))).half()
    got = P.context_attention(q.cuda(), dev_pages(pages, hd), table.cuda(), i32([n]).cuda(), 1).cpu()
    k = pages[0].reshape(-1, R.width(hd))[:n, :hd].double()
    v = pages[1].permute(0, 3, 1, 2).reshape(-1, R.width(hd))[:n, :hd].double()
    p = torch.softmax(k @ q[0, 0].double() * hd ** -0.5, 0)
    want, size = p @ v, float((k.abs() @ q[0, 0].double().abs()).max()) * hd ** -0.5
    # the bound of paged_reference.attention
    rel = 2 * (hd + 4) * R.U * size + (n + 8) * R.U + 2.0 ** -16 + n * 2.0 ** -31
    bound = 2 * rel * (p @ v.abs()) + R.HALF_STEP[torch.float16] * want.abs() * (1 + rel) + 2.0 ** -25
    assert bool(((got[0, 0].double() - want).abs() <= bound).all())


def test_attention_skips_pages_that_are_not_there():
    pages = R.make_pages(5, 1, 16, 16, torch.float32)
    table = i32([[0, -1, 7, 3, 1], [-1, -1, 9, 5, -3]])
    q = torch.randn(2, 1, 16)
    lengths = [75, 80]
    got = P.context_attention(q.cuda(), dev_pages(pages, 16), table.cuda(), i32(lengths).cuda(), 1).cpu()
    want, bound = R.attention(q, pages, table, lengths, 1, 16)
    assert bool(((got.double() - want).abs() <= bound).all()) and float(got[1].abs().max()) == 0.0
    # lengths outside what the table holds are clamped
    for n, m in ((2 ** 31 - 1, 80), (-5, 0)):
        got = P.context_attention(q.cuda(), dev_pages(pages, 16), table.cuda(), i32([n, n]).cuda(), 1).cpu()
        want, bound = R.attention(q, pages, table, [m, m], 1, 16)
        assert bool(((got.double() - want).abs() <= bound).all())


def test_attention_of_extreme_logits():
    """Logits hundreds apart: the running maximum moves, all but the largest weights vanish, nothing overflows."""
    hd, n = 32, 400
    for dtype in DTYPES:
        pages = R.make_pages(7, 1, 64, hd, dtype, 4)
        table = i32([list(range(7))])
        for p in range(7):
            pages[0][p] *= 40.0 * (1 if p % 2 else -1)
        q = (4 * torch.randn(1, 3, hd, generator=torch.Generator().manual_seed(8))).to(dtype)
        got = P.context_attention(q.cuda(), dev_pages(pages, hd), table.cuda(), i32([n]).cuda(), 1).cpu()
        want, bound = R.attention(q, pages, table, [n], 1, hd)
        assert bool(((got.double() - want).abs() <= bound).all()), dtype


# ---- selection -----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("heads,kv,hd,page,T,lengths,count", [
    (8, 8, 15, 32, 2, [700, 1, 0, 33], 5),
    (8, 2, 64, 16, 1, [999, 16, 17], 16),
    (6, 1, 128, 64, 3, [64 * 9 + 1], 100),
    (2, 2, 7, 16, 1, [16 * 1500], 129),
    (4, 2, 250, 16, 1, [300], 1),
    (40, 2, 33, 16, 2, [211], 3),
])
def test_selection(dtype, heads, kv, hd, page, T, lengths, count):
    need = [-(-n // page) for n in lengths]
    pool = sum(need) + 2
    pages = R.make_pages(pool, kv, page, hd, dtype, 9)
    table = R.make_table(need, max(need) + 2, pool, 9)
    table[0, min(3, table.shape[1] - 1)] = -1 if count % 2 else pool
    q = torch.randn(len(lengths), T, heads * hd, generator=torch.Generator().manual_seed(9)).to(dtype)
    got = P.select_pages(q.cuda(), dev_pages(pages, hd), table.cuda(), i32(lengths).cuda(), heads, count)
    assert torch.equal(got.cpu(), R.select(q, pages[2], pages[3], table, lengths, page, heads, hd, count))


def test_selection_takes_the_lower_page_among_equals():
    pages = R.make_pages(40, 1, 16, 16, torch.bfloat16, 2)
    low, high = pages[2].clone(), pages[3].clone()
    low[:], high[:] = low[0], high[0]  # all alike ...
    low[7], high[7] = -9.0, 9.0        # ... but two better and one worse
    low[21], high[21] = -9.0, 9.0
    low[2], high[2] = 0.0, 0.0
    q = torch.randn(1, 1, 16, generator=torch.Generator().manual_seed(1)).bfloat16()
    table = torch.arange(40, dtype=torch.int32)[None].contiguous()
    got = P.select_pages(q.cuda(), P.ContextPages(pages[0].cuda(), pages[1].cuda(), low.cuda(), high.cuda(), 16), table.cuda(), i32([640]).cuda(), 1, 8)
    assert got.flatten().tolist() == [0, 1, 3, 4, 5, 6, 7, 21]
    low[30, 0, 0] = math.nan  # a page whose score is not a number comes first
    got = P.select_pages(q.cuda(), P.ContextPages(pages[0].cuda(), pages[1].cuda(), low.cuda(), high.cuda(), 16), table.cuda(), i32([640]).cuda(), 1, 2)
    assert got.flatten().tolist() == [7, 30]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("pages,count", [(60, 20), (1500, 700), (5000, 33)])
def test_selection_between_scores_that_32_bits_do_not_tell_apart(dtype, pages, count):
    """One large product that every page has, and differences far below its rounding: the order is that of 64 bits."""
    hd, g = 16, torch.Generator().manual_seed(pages)
    low = torch.zeros(pages, 1, 16, dtype=dtype)
    high = torch.zeros(pages, 1, 16, dtype=dtype)
    high[:, 0, 0] = 2048.0
    high[:, 0, 1:4] = (torch.randint(0, 200, (pages, 3), generator=g) / 256.0).to(dtype)
    low[:, 0, 4] = (-torch.randint(0, 3, (pages,), generator=g) / 64.0).to(dtype)
    q = torch.zeros(1, 1, hd, dtype=dtype)
    q[0, 0, :5] = torch.tensor([1024.0, 2.0 ** -9, 2.0 ** -8, 2.0 ** -10, -(2.0 ** -12)]).to(dtype)
    keys, values = torch.zeros(pages, 1, 16, 16, dtype=dtype), torch.zeros(pages, 1, 16, 16, dtype=dtype)
    table = torch.randperm(pages, generator=g).to(torch.int32)[None].contiguous()
    context = P.ContextPages(keys.cuda(), values.cuda(), low.cuda(), high.cuda(), hd)
    got = P.select_pages(q.cuda(), context, table.cuda(), i32([16 * pages]).cuda(), 1, count)
    assert torch.equal(got.cpu(), R.select(q, low, high, table, [16 * pages], 16, 1, hd, count))
    # a query of zeros: every page scores zero, the first ones are taken
    got = P.select_pages(torch.zeros_like(q).cuda(), context, table.cuda(), i32([16 * pages]).cuda(), 1, count)
    assert got.flatten().tolist() == list(range(count))


@pytest.mark.parametrize("pages,count", [(1536, 100), (1537, 100), (8192, 4000), (8193, 300), (9000, 2000), (40000, 100), (31251, 128), (40000, 300), (40000, 1000), (40000, 39999)])
def test_selection_from_long_rows(pages, count):
    """Rows that one workgroup takes, with its buckets in LDS or beyond them, and rows cut into segments; then a few scores far out that
    squeeze all others into one bucket, and a query of zeros."""
    hd = 16
    g = torch.Generator().manual_seed(4)
    low = torch.randn(pages, 1, 16, generator=g) - 1
    high = low + torch.rand(pages, 1, 16, generator=g)
    q = torch.randn(1, 1, hd, generator=g)
    table = torch.arange(pages, dtype=torch.int32)[None].contiguous()
    keys = torch.zeros(pages, 1, 16, 16)
    for far in (None, 1e30):
        if far:
            high[[7, pages - 1], 0, 0] = far
            low[[7, pages - 1], 0, 0] = -far
        context = P.ContextPages(keys.cuda(), keys.cuda(), low.cuda(), high.cuda(), hd)
        got = P.select_pages(q.cuda(), context, table.cuda(), i32([16 * pages - 3]).cuda(), 1, count)
        exact = (q.double().clamp(min=0) * high[:, 0].double() + q.double().clamp(max=0) * low[:, 0].double()).sum(-1).flatten()
        want = torch.sort(torch.sort(exact, descending=True, stable=True).indices[:count]).values.int()
        assert torch.equal(got.cpu().flatten(), want)
    got = P.select_pages(torch.zeros_like(q).cuda(), context, table.cuda(), i32([16 * pages]).cuda(), 1, count)
    assert got.flatten().tolist() == list(range(count))


# ---- together ------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_growing_contexts(dtype):
    """Contexts grow step by step (none, one, many tokens); after each step attention equals attention over all tokens so far, and the
    selection of every page, or of more than there are, equals it too."""
    heads, hd, page, B = 4, 16, 16, 3
    context = P.allocate_pages(24, heads, hd, page, dtype)
    table = R.make_table([8, 8, 8], 8, 24, 1)
    held = [0, 0, 0]
    g = torch.Generator().manual_seed(2)
    for counts in ([3, 0, 40], [1, 1, 1], [0, 17, 16], [14, 1, 0], [1, 0, 71]):
        n = sum(counts)
        k, v = (torch.randn(n, heads * hd, generator=g).to(dtype) for _ in range(2))
        xyz = torch.rand(n, 2, generator=g)
        offsets = i32([0] + torch.tensor(counts).cumsum(0).tolist())
        P.append_context(context, k.cuda(), v.cuda(), offsets.cuda(), i32(held).cuda(), table.cuda(), xyz.cuda(), hd)
        held = [a + b for a, b in zip(held, counts)]
        q = torch.randn(B, 2, heads * hd, generator=g).to(dtype)
        pages = [t.cpu() for t in context[:4]]
        want, bound = R.attention(q, pages, table, held, heads, hd)
        got = P.context_attention(q.cuda(), context, table.cuda(), i32(held).cuda(), heads)
        assert bool(((got.cpu().double() - want).abs() <= bound).all())
        chosen = P.select_pages(q.cuda(), context, table.cuda(), i32(held).cuda(), heads, 9)
        got = P.context_attention(q.cuda(), context, table.cuda(), i32(held).cuda(), heads, pages=chosen)
        assert bool(((got.cpu().double() - want).abs() <= bound).all())


def test_no_contexts_and_no_tokens():
    context = P.allocate_pages(2, 2, 16, 16)
    none = torch.zeros(0, 32).cuda()
    P.append_context(context, none, none, i32([0, 0]).cuda(), i32([0]).cuda(), i32([[0, 1]]).cuda())
    P.append_context(context, none, none, i32([0]).cuda(), i32([]).cuda(), torch.zeros(0, 2, dtype=torch.int32).cuda())
    assert P.context_attention(torch.zeros(0, 1, 32).cuda(), context, torch.zeros(0, 2, dtype=torch.int32).cuda(), i32([]).cuda(), 2).shape == (0, 1, 32)
    out = P.context_attention(torch.ones(1, 1, 32).cuda(), context, torch.zeros(1, 0, dtype=torch.int32).cuda(), i32([5]).cuda(), 2)
    assert float(out.abs().max()) == 0.0
    assert P.select_pages(torch.ones(1, 1, 32).cuda(), context, torch.zeros(1, 0, dtype=torch.int32).cuda(), i32([5]).cuda(), 2, 3).flatten().tolist() == [-1] * 6


def test_captured_calls_replay_with_other_lengths():
    """Two graphs of append + selection + attention on their own streams' workspaces, replayed in turn with eager calls between."""
    heads, hd, page, dtype = 4, 32, 16, torch.bfloat16
    context = P.allocate_pages(130, heads, hd, page, dtype)
    table = R.make_table([64, 64], 64, 130, 3).cuda()
    g = torch.Generator().manual_seed(4)
    kv = torch.randn(400, 2 * heads * hd, generator=g).to(dtype).cuda()
    starts, offsets, lengths = i32([0, 0]).cuda(), i32([0, 0, 0]).cuda(), i32([0, 0]).cuda()
    positions = torch.rand(400, 1, generator=g).cuda()
    q = torch.randn(2, 3, heads * hd, generator=g).to(dtype).cuda()

    def step():
        P.append_context(context, kv[:, :heads * hd], kv[:, heads * hd:], offsets, starts, table, positions, hd)
        chosen = P.select_pages(q, context, table, lengths, heads, 7)
        return P.context_attention(q, context, table, lengths, heads), chosen, P.context_attention(q, context, table, lengths, heads, pages=chosen)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    held = [0, 0]
    for i, counts in enumerate(([17, 300], [1, 0], [0, 64], [200, 200], [33, 1])):
        starts.copy_(i32(held))
        offsets.copy_(i32([0, counts[0], counts[0] + counts[1]]))
        held = [a + b for a, b in zip(held, counts)]
        lengths.copy_(i32(held))
        q.copy_(torch.randn(2, 3, heads * hd, generator=g).to(dtype))
        graph, out = graphs[i % 2]
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in out]
        eager = step()
        torch.cuda.synchronize()
        for a, b in zip(replayed, eager):
            assert torch.equal(a, b)
        want, bound = R.attention(q.cpu(), [t.cpu() for t in context[:4]], table.cpu(), held, heads, hd)
        assert bool(((eager[0].cpu().double() - want).abs() <= bound).all())


def test_on_another_stream():
    context = P.ContextPages(*(t.cuda() for t in R.make_pages(20, 2, 16, 16, torch.float32)), 16)
    table = torch.arange(20, dtype=torch.int32).cuda()[None].contiguous()
    q = torch.randn(1, 1, 32).cuda()
    lengths = i32([300]).cuda()
    want = P.context_attention(q, context, table, lengths, 2)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = P.context_attention(q, context, table, lengths, 2)
        chosen = P.select_pages(q, context, table, lengths, 2, 30)
    side.synchronize()
    assert torch.equal(got, want) and (chosen >= 0).sum() == 2 * 19


def test_pools_beyond_32_bit_offsets():
    """Pages whose first element is beyond 2^32 elements of the pool."""
    heads, hd, page = 1, 128, 256
    num = 2 ** 32 // (page * 128) + 40  # 8.6 GB of keys, 8.6 GB of values
    context = P.allocate_pages(num, heads, hd, page, torch.bfloat16)
    ids = [num - 1, 3, num - 7, num // 2 + 5]
    table = i32([ids])
    g = torch.Generator().manual_seed(1)
    n = 4 * page - 9
    k, v = (torch.randn(n, hd, generator=g).bfloat16() for _ in range(2))
    P.append_context(context, k.cuda(), v.cuda(), i32([0, n]).cuda(), i32([0]).cuda(), table.cuda())
    at = torch.tensor(ids).cuda()
    small = [context.keys[at].cpu(), context.values[at].cpu()]
    assert torch.equal(small[0].reshape(-1, hd)[:n], k) and torch.equal(small[1].permute(0, 3, 1, 2).reshape(-1, hd)[:n], v)
    q = torch.randn(1, 1, hd, generator=g).bfloat16()
    got = P.context_attention(q.cuda(), context, table.cuda(), i32([n]).cuda(), 1)
    want, bound = R.attention(q, small, i32([[0, 1, 2, 3]]), [n], 1, hd)
    assert bool(((got.cpu().double() - want).abs() <= bound).all())
    chosen = P.select_pages(q.cuda(), context, table.cuda(), i32([n]).cuda(), 1, 2)
    assert torch.equal(chosen.cpu(), R.select(q, context.key_min[at].cpu(), context.key_max[at].cpu(), i32([[0, 1, 2, 3]]), [n], page, 1, hd, 2))


def test_repeated_calls_give_the_same_bits():
    context = P.ContextPages(*(t.cuda() for t in R.make_pages(400, 2, 32, 64, torch.float16)), 64)
    table = torch.randperm(400, generator=torch.Generator().manual_seed(0)).to(torch.int32).cuda()[None].contiguous()
    q = torch.randn(1, 4, 8 * 64).half().cuda()
    first = P.context_attention(q, context, table, i32([12700]).cuda(), 8)
    for _ in range(3):
        assert torch.equal(P.context_attention(q, context, table, i32([12700]).cuda(), 8), first)
