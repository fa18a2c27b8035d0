"""The paged context operators at the edges of what their documentation allows: rows that are taken whole, scores that are not numbers,
lengths far outside the table, launch forms of large calls (against the 64-bit restatement of paged_reference)."""
import math

import math

import pytest
import torch

import paged_reference as R
from nvblox_mindmap_amd.diffuser_actor import paged_context as P

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def summaries(low, high, hd, page=16):
    """Pages [n, kv_heads, 16] that only a selection reads: their summaries, and keys / values that may be any."""
    n, heads, w = low.shape
    empty = torch.zeros((n, heads, page, w), dtype=low.dtype, device="cuda")
    return P.ContextPages(empty, torch.zeros((n, heads, w, page), dtype=low.dtype, device="cuda"), low.cuda(), high.cuda(), hd)


# slots of the table, pages that a context holds, count: every launch form of the selection (four waves, sixteen, segments, a row of any
# length), each with more entries than threads and a count that takes them all
@pytest.mark.parametrize("slots,held,count", [(1536, 257, 512), (1536, 400, 400), (700, 700, 701), (1536, 1536, 1536), (8192, 1100, 1100), (5000, 4999, 6000), (8192, 8192, 8192),
                                              (40000, 100, 128), (8193, 1365, 1365), (40000, 409, 409), (40000, 5000, 5000), (40000, 40000, 40000)])
def test_a_row_that_is_taken_whole(slots, held, count):
    """As many pages as the context holds, or more: all of them in order, then -1, whatever the signs of their scores."""
    H, T, hd, pool = 4, 2, 16, 64
    g = torch.Generator().manual_seed(slots + held)
    low = -torch.rand(pool, H, 16, generator=g) - 1.0
    q = torch.rand(2, T, H * hd, generator=g) + 0.1  # scores of -1.6 to -36
    q[1, 1] *= torch.where(torch.rand(H * hd, generator=g) < 0.5, 1.0, -1.0)  # ... and of both signs
    table = torch.randint(0, pool, (2, slots), generator=g).to(torch.int32)
    table[1, ::5] = -1
    lengths = i32([16 * held - 15, 16 * held])
    got = P.select_pages(q.cuda(), summaries(low, low * 0.9, hd), table.cuda(), lengths.cuda(), H, count).cpu()
    for b in range(2):
        there = (table[b, :held] >= 0).nonzero().flatten().to(torch.int32)
        want = torch.cat([there, torch.full((count - len(there),), -1, dtype=torch.int32)])
        assert torch.equal(got[b], want.expand(T, H, count)), b


# pages, how many of them have no number for a score, how many share the largest score, count
@pytest.mark.parametrize("pages,nans,tops,count", [(1000, 300, 1, 7), (1000, 300, 1, 300), (1000, 300, 1, 299), (1000, 300, 1, 500), (700, 5, 300, 2), (700, 5, 300, 5), (700, 5, 300, 6), (700, 5, 300, 400),
                                                   (5000, 600, 2, 333), (5000, 3, 900, 3), (40000, 2000, 1, 100), (40000, 5000, 300, 4500), (40000, 9, 5000, 8), (40000, 9, 9000, 5000)])
def test_pages_whose_score_is_not_a_number_come_first(pages, nans, tops, count):
    """Several hundred of them, or of the largest number, share the bucket that holds the border: it is divided again, up to the very end of the keys' range."""
    hd, g = 16, torch.Generator().manual_seed(pages + nans)
    high = torch.rand(pages, 1, 16, generator=g)
    q = torch.rand(1, 1, hd, generator=g) + 0.1
    place = torch.randperm(pages - 1, generator=g) + 1
    best = torch.cat([torch.zeros(1, dtype=torch.long), place[:tops - 1]])  # slot 0 among them
    high[best] = 1.5
    none = place[tops:tops + nans]
    high[none, 0, 3] = math.nan
    table = torch.arange(pages, dtype=torch.int32)[None].contiguous()
    got = P.select_pages(q.cuda(), summaries(high, high, hd), table.cuda(), i32([16 * pages]).cuda(), 1, count).cpu().flatten()
    score = (q.double() * high[:, 0].double()).sum(-1).flatten()
    order = torch.sort(torch.where(torch.isnan(score), math.inf, score), descending=True, stable=True).indices
    assert torch.equal(got, torch.sort(order[:count]).values.int())


@pytest.mark.parametrize("n", [-2 ** 31, -2 ** 31 + 1, -2 ** 31 + 47, -5, 2 ** 31 - 1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_lengths_far_outside_the_table(n, dtype):
    """A length is clamped to what the table holds, on every path; below zero there is no token."""
    pages = R.make_pages(6, 2, 16, 16, dtype)
    table, q = i32([[2, 4, 0, 1, 5]]), torch.randn(1, 2, 32, generator=torch.Generator().manual_seed(1)).to(dtype)
    context = P.ContextPages(*(t.cuda() for t in pages), 16)
    lengths, held = i32([n]).cuda(), 0 if n < 0 else 80
    selected = i32([0, 1, 3, 4]).expand(1, 2, 2, 4).contiguous()
    for chosen in (None, selected):
        got = P.context_attention(q.cuda(), context, table.cuda(), lengths, 2, pages=None if chosen is None else chosen.cuda()).cpu()
        want, bound = R.attention(q, pages, table, [held], 2, 16, selected=chosen)
        assert bool(((got.double() - want).abs() <= bound).all())
    got = P.select_pages(q.cuda(), context, table.cuda(), lengths, 2, 3).cpu()
    assert torch.equal(got, R.select(q, pages[2], pages[3], table, [held], 16, 2, 16, 3))


@pytest.mark.parametrize("kind", ["gradient", "tangent"])
def test_inputs_with_derivatives_are_refused(kind):
    """No operator loses a gradient or a tangent in silence: of the query, the rows, the positions, or the pages themselves."""
    from torch.autograd import forward_ad

    def mark(t):
        return t.clone().requires_grad_() if kind == "gradient" else forward_ad.make_dual(t.clone(), torch.ones_like(t))

    table, lengths, offsets = i32([[0, 1]]).cuda(), i32([20]).cuda(), i32([0, 3]).cuda()
    q, rows, positions = torch.randn(1, 1, 32).cuda(), torch.randn(3, 32).cuda(), torch.rand(3, 1).cuda()
    context = P.ContextPages(*(t.cuda() for t in R.make_pages(2, 2, 16, 16, torch.float32)), 16)
    with forward_ad.dual_level():
        marked = [context._replace(keys=mark(context.keys)), context._replace(values=mark(context.values))]
        calls = [lambda: P.context_attention(mark(q), context, table, lengths, 2), lambda: P.select_pages(mark(q), context, table, lengths, 2, 1),
                 lambda: P.append_context(context, mark(rows), rows, offsets, lengths, table), lambda: P.append_context(context, rows, mark(rows), offsets, lengths, table),
                 lambda: P.append_context(context, rows, rows, offsets, lengths, table, mark(positions))]
        calls += [lambda c=c: P.context_attention(q, c, table, lengths, 2) for c in marked]
        calls += [lambda c=c: P.append_context(c, rows, rows, offsets, lengths, table) for c in marked]
        for call in calls:
            with pytest.raises(RuntimeError, match="no backward"):
                call()
        assert bool(torch.isfinite(P.context_attention(q, context, table, lengths, 2)).all())
    with torch.no_grad():
        if kind == "gradient":
            assert not P.context_attention(mark(q), context, table, lengths, 2).requires_grad


def mesh_model(seed=0):
    from nvblox_mindmap_amd.diffuser_actor import DiffuserActor, DiffuserActorConfig

    torch.manual_seed(seed)
    model = DiffuserActor(DiffuserActorConfig(data_type="mesh", feature_dim=16, diffusion_timesteps=3), torch.tensor([[-1.0, -1, -1], [1, 1, 1]]))
    return model.cuda().eval()


def mesh_observation(seed, batch=2, n=120):
    """Arguments of DiffuserActor.forward."""
    g = torch.Generator().manual_seed(seed)
    pose = torch.cat([torch.rand(batch, 3, 2, 3, generator=g), torch.nn.functional.normalize(torch.randn(batch, 3, 2, 4, generator=g), dim=-1), torch.ones(batch, 3, 2, 1)], -1)
    return [None] * 5 + [torch.randn(batch, n, 16, generator=g).cuda(), (torch.rand(batch, n, 3, generator=g) * 1.8 - 0.9).cuda(),
                         (torch.rand(batch, n, generator=g) > 0.3).cuda(), None, pose.cuda()]


@pytest.mark.parametrize("autocast", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@torch.no_grad()
def test_the_policy_keeps_a_memory_under_autocast(autocast, dtype):
    model = mesh_model()
    memory = model.new_context_memory(2, 32, 16, dtype)
    one, two = mesh_observation(1), mesh_observation(2)
    with torch.autocast("cuda", autocast):
        for args in (one, two):
            assert bool(torch.isfinite(model(*args, run_inference=True, context_memory=memory)[0]).all())
    assert memory.held == tuple((one[7].sum(1) + two[7].sum(1)).tolist())


@pytest.mark.parametrize("on", [False, True], ids=["composite", "fused"])
@torch.no_grad()
def test_a_robot_that_has_seen_nothing(on):
    """A sample without a valid context token attends, without a memory, to zeroed tokens, whose values are the projection's bias; a memory
    that holds nothing of it gives the same."""
    from nvblox_mindmap_amd.diffuser_actor import DiffuserActor

    model = mesh_model()
    for name, p in model.named_parameters():  # as a trained model has them
        if name.endswith("kv_proj.bias"):
            torch.nn.init.normal_(p, std=0.5)
        if name.endswith("adaln.proj.weight"):
            torch.nn.init.normal_(p, std=0.05)
    args = mesh_observation(5)
    args[7][1] = False
    memory = model.new_context_memory(2, 32, 16)
    DiffuserActor.enable_fused_inference(on)
    try:
        torch.manual_seed(3)
        plain = model(*args, run_inference=True)[0]
        torch.manual_seed(3)
        kept = model(*args, run_inference=True, context_memory=memory)[0]
        # two float32 evaluations of a denoising loop of three steps, positions in metres (as between the two evaluations of a full context)
        assert float((plain - kept)[..., :3].abs().max()) <= 5e-3
        stack, query, cond = model.prediction_head.cross_attn, torch.randn(2, 4, 120).cuda(), torch.randn(2, 120).cuda()
        nothing = torch.zeros(2, 1, 120).cuda()
        want = stack(query, nothing, cond)[0][1]
        # 32-bit evaluations of one layer's worth of sums of 120 products, through two layers with a gain of a few each
        assert float((stack(query, None, cond, kv_caches=memory.layers)[0][1] - want).abs().max()) <= 2e-4
        # captured: an empty context may have tokens, or lose them, between replays
        graph = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            stack(query, None, cond, kv_caches=memory.layers)
        torch.cuda.current_stream().wait_stream(side)
        with torch.cuda.graph(graph):
            out = stack(query, None, cond, kv_caches=memory.layers)[0]
        for step in range(3):
            if step == 1:
                memory.release(0)
            elif step == 2:
                rows = torch.randn(40, 120).cuda()
                memory.append([0, 40], [(rows, rows)] * 2)
            graph.replay()
            assert torch.equal(out, stack(query, None, cond, kv_caches=memory.layers)[0]), step
            if step == 1:
                assert float((out - stack(query, nothing, cond)[0]).abs().max()) <= 2e-4
    finally:
        DiffuserActor.enable_fused_inference(False)


# ---- launch forms of large calls ----
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("hd", [15, 80, 128, 250])  # widths 16, 96, 128, 256
@pytest.mark.parametrize("rows,n", [(17, 5003), (33, 3001), (40, 4099), (17, 20005), (33, 18000)])  # at most 64 splits, and more
def test_many_rows_over_split_contexts(dtype, hd, rows, n):
    """17 and more query rows of a key-value head -- two row tiles, several row blocks -- whose partial results are joined; as query tokens, as
    heads that share the keys, and as such heads over selected pages."""
    page, g = 256, torch.Generator().manual_seed(rows + n)
    need = -(-n // page)
    pages = R.make_pages(need, 1, page, hd, dtype, n)
    table = R.make_table([need], need + 1, need, n)
    context, lengths = P.ContextPages(*(t.cuda() for t in pages), hd), i32([n]).cuda()
    at = table[0, :need].long()
    k = pages[0][at, 0, :, :hd].reshape(-1, hd)[:n].double()
    v = pages[1][at, 0, :hd].permute(0, 2, 1).reshape(-1, hd)[:n].double()
    x = (1.5 * torch.randn(rows, hd, generator=g)).to(dtype)
    slots = torch.randperm(need + 1, generator=g)[:need - 2].to(torch.int32)  # (the last slot of the table has no page)
    place = torch.arange(n) // page
    for q, heads, chosen in ((x.view(1, rows, hd), 1, None), (x.view(1, 1, rows * hd), rows, None), (x.view(1, 1, rows * hd), rows, slots)):
        kk, vv = (k, v) if chosen is None else (k[torch.isin(place, chosen.long())], v[torch.isin(place, chosen.long())])
        got = P.context_attention(q.cuda(), context, table.cuda(), lengths, heads, pages=None if chosen is None else chosen.view(1, 1, 1, -1).cuda()).cpu()
        xd = x.double()
        p = torch.softmax(xd @ kk.T * hd ** -0.5, 1)
        want, size = p @ vv, (xd.abs() @ kk.abs().T).amax(1, keepdim=True) * hd ** -0.5
        # the bound of paged_reference.attention
        rel = 2 * (hd + 4) * R.U * size + (len(kk) + 8) * R.U + (0.0 if dtype == torch.float32 else 2.0 ** -16 + len(kk) * 2.0 ** -31)
        bound = 2 * rel * (p @ vv.abs()) + R.HALF_STEP[dtype] * want.abs() * (1 + rel) + 2.0 ** -25 * (dtype == torch.float16)
        off = (got.view(rows, hd).double() - want).abs()
        assert bool((off <= bound).all()), (heads, chosen is not None, float((off / bound).max()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("hd,batch,kv,slots", [(250, 8, 16, 531), (128, 8, 16, 1060), (80, 16, 16, 530), (64, 16, 12, 1400), (16, 16, 16, 4100), (128, 16, 16, 8200)])
@pytest.mark.parametrize("tokens,group", [(1, 1), (2, 4), (3, 3), (1, 17)])
def test_scores_of_many_pages(dtype, hd, batch, kv, slots, tokens, group):
    """Workgroups that score several sets of pages one after the other (up to 16), with eight query rows a key-value head and with more; the
    same pages stand in many slots, so equal scores abound."""
    pool, page, count, g = 96, 16, 9, torch.Generator().manual_seed(hd + slots)
    pages = R.make_pages(pool, kv, page, hd, dtype, hd)
    table = torch.randint(-1, pool, (batch, slots), generator=g).to(torch.int32)
    held = torch.randint(1, slots + 1, (batch,), generator=g)
    held[0], held[1] = slots, 0
    q = torch.randn(batch, tokens, kv * group * hd, generator=g).to(dtype)
    got = P.select_pages(q.cuda(), P.ContextPages(*(t.cuda() for t in pages), hd), table.cuda(), (held * page).to(torch.int32).cuda(), kv * group, count).cpu()
    x = q.double().view(batch, tokens, kv, group, hd).permute(2, 0, 1, 3, 4).reshape(kv, -1, hd)
    low, high = (t[..., :hd].double().permute(1, 2, 0).contiguous() for t in (pages[2], pages[3]))
    score = (torch.matmul(x.clamp(min=0), high) + torch.matmul(x.clamp(max=0), low)).view(kv, batch, tokens, group, pool).amax(3)
    for b in range(batch):
        there = (torch.arange(slots) < held[b]) & (table[b] >= 0)
        s = score[:, b][..., table[b].clamp(min=0).long()].masked_fill(~there, -math.inf)  # [kv, tokens, slots]
        order = torch.sort(s, dim=-1, descending=True, stable=True).indices[..., :count]
        order = torch.where(torch.gather(s, 2, order) > -math.inf, order, slots).sort(-1).values
        want = torch.where(order < slots, order, -1).to(torch.int32)
        assert torch.equal(got[b], want.transpose(0, 1)), b


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("selected", [None, 2])
@torch.no_grad()
def test_a_memory_in_16_bits_is_that_of_its_rounded_keys_and_values(dtype, selected):
    """Two observations through the policy's projections: the pages hold them rounded once, and a layer's attention is that of the rounded
    query over them."""
    head = mesh_model(1).prediction_head
    memory = P.ContextMemory(2, 2, 16, 8, 15, 16, dtype, selected_pages=selected)
    g, seen = torch.Generator().manual_seed(7), [[], []]
    for sizes in ((40, 7), (23, 30)):
        n = max(sizes)
        mask = torch.arange(n)[None] < torch.tensor(sizes)[:, None]
        enc = {"context_feats": torch.randn(2, n, 120, generator=g).cuda(), "context_pos": (torch.rand(2, n, 3, generator=g) * 2 - 1).cuda(), "context_mask": mask.cuda()}
        head.extend_memory(memory, enc)
        for b, m in enumerate(sizes):
            seen[b].append((enc["context_feats"][b, :m], enc["context_pos"][b, :m].cpu()))
    t = memory.pages_of
    assert t.held == (63, 37)
    for layer, blk in zip(memory.layers, head.cross_attn.attn):
        pages = [x.cpu() for x in layer.pages[:4]]
        for b in range(2):
            for h in range(8):
                k, v, _ = R.context(pages, t.table[b].cpu(), t.held[b], h, 15)
                start = 0
                for f, xyz in seen[b]:
                    kv = blk.attn.kv_proj(f).cpu().double()
                    rotated = R.rotate(kv[:, :120], xyz, None, 8, 15)[:, 15 * h:15 * h + 15]
                    for got, want in ((k, rotated), (v, kv[:, 120 + 15 * h:135 + 15 * h])):
                        # the rounding to the pages' type; rotation in 32 bits, and the projection of more rows at once: sums of 120 products in another order
                        slack = (12 * 2 + 2 * 120) * R.U * float(kv.abs().max()) * 2 + 2.0 ** -25 * (dtype == torch.float16)
                        assert bool(((got[start:start + len(f)] - want).abs() <= R.HALF_STEP[dtype] * want.abs() + slack).all())
                    start += len(f)
        q = torch.randn(2, 3, 120, generator=g)
        chosen = None if selected is None else R.select(q.to(dtype), pages[2], pages[3], t.table.cpu(), t.held, 16, 8, 15, selected)
        want, bound = R.attention(q.to(dtype), pages, t.table.cpu(), t.held, 8, 15, selected=chosen)
        got = layer.attend(q.cuda(), 8, blk.attn.empty_value())
        assert got.dtype == torch.float32 and bool(((got.cpu().double() - want).abs() <= bound).all())
