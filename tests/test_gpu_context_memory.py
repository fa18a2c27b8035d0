"""The policy's cross-attention over a paged context memory (paged_context.ContextMemory, DiffuserActor.forward(context_memory=))."""
import pytest
import torch

from nvblox_mindmap_amd.diffuser_actor import DiffuserActor, DiffuserActorConfig, layers as L
from nvblox_mindmap_amd.diffuser_actor import paged_context as P

pytestmark = pytest.mark.gpu
D, H = 120, 8
# Two float32 evaluations of the same stack: logits and weighted sums over a few hundred keys differ by at most some 300 roundings (2e-5 of
# values of size one), which two projections with row norms of about one and a LayerNorm of rows with deviation of about one pass on with a
# gain of a few, twice.
STACK = 2e-4


@pytest.fixture
def fused():
    yield DiffuserActor.enable_fused_inference
    DiffuserActor.enable_fused_inference(False)


def make_stack(seed=0):
    torch.manual_seed(seed)
    stack = L.AttentionStack(D, H, 2, use_adaln=True).cuda().eval()
    for p in stack.parameters():
        if p.dim() == 2 and float(p.detach().abs().max()) == 0.0:  # AdaLN starts as the identity: make it count
            torch.nn.init.normal_(p, std=0.05)
    return stack


def observation(n, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(n, D, generator=g).cuda(), (torch.rand(n, 3, generator=g) * 2 - 1).cuda()


def remember(stack, memory, observations):
    """observations: one (features, positions) per context."""
    feats, pos = torch.cat([f for f, _ in observations]), torch.cat([p for _, p in observations]).contiguous()
    memory.append([f.shape[0] for f, _ in observations], [b.attn.project_paged(feats) for b in stack.attn], pos, D)


def dense(stack, query, cond, q_rot, contexts):
    """The stack over padded contexts with a mask."""
    n = max(f.shape[0] for f, _ in contexts)
    feats, pos, pad = torch.zeros(len(contexts), n, D).cuda(), torch.zeros(len(contexts), n, 3).cuda(), torch.ones(len(contexts), n, dtype=torch.bool).cuda()
    for b, (f, p) in enumerate(contexts):
        feats[b, :len(f)], pos[b, :len(f)], pad[b, :len(f)] = f, p, False
    return stack(query, feats, cond, q_rot, L.rotary3d(pos, D), key_padding_mask=pad)[0]


@pytest.mark.parametrize("on", [False, True], ids=["composite", "fused"])
@pytest.mark.parametrize("tokens", [1, 2, 17])
@torch.no_grad()
def test_memory_is_the_concatenation_of_its_observations(fused, on, tokens):
    stack = make_stack()
    memory = P.ContextMemory(2, 3, 64, H, 15, 32)
    seen = [[], [], []]
    g = torch.Generator().manual_seed(5)
    for step, sizes in enumerate(([70, 1, 200], [33, 64, 7], [1, 90, 0])):
        new = [observation(n, 10 * step + b) for b, n in enumerate(sizes)]
        fused(False)
        remember(stack, memory, new)
        for b in range(3):
            seen[b].append(new[b])
        contexts = [(torch.cat([f for f, _ in s]), torch.cat([p for _, p in s])) for s in seen]
        query, cond = torch.randn(3, tokens, D, generator=g).cuda(), torch.randn(3, D, generator=g).cuda()
        q_rot = L.rotary3d((torch.rand(3, tokens, 3, generator=g) * 2 - 1).cuda(), D)
        want = dense(stack, query, cond, q_rot, contexts)
        fused(on)
        got, weights = stack(query, None, cond, q_rot, None, kv_caches=memory.layers)
        assert weights is None and float((got - want).abs().max()) <= STACK
    assert memory.held == (104, 155, 207)


@torch.no_grad()
def test_released_pages_serve_another_context(fused):
    stack = make_stack(1)
    memory = P.ContextMemory(2, 2, 8, H, 15, 16)
    first, second = observation(100, 1), observation(120, 2)
    none = (torch.zeros(0, D).cuda(), torch.zeros(0, 3).cuda())
    remember(stack, memory, [first, none])
    with pytest.raises(RuntimeError, match="free"):
        remember(stack, memory, [none, second])
    assert memory.held == (100, 0)
    memory.release(0)
    remember(stack, memory, [none, second])
    query, cond = torch.randn(2, 2, D).cuda(), torch.randn(2, D).cuda()
    q_rot = L.rotary3d(torch.rand(2, 2, 3).cuda(), D)
    got = stack(query, None, cond, q_rot, None, kv_caches=memory.layers)[0]
    want = dense(stack, query[1:], cond[1:], (q_rot[0][1:], q_rot[1][1:]), [second])
    assert float((got[1:] - want).abs().max()) <= STACK and bool(torch.isfinite(got).all())  # context 0 is empty: attention of zeros


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@torch.no_grad()
def test_selecting_every_page_is_attending_to_all(dtype):
    stack = make_stack(2)
    memory = P.ContextMemory(2, 1, 16, H, 15, 16, dtype)
    remember(stack, memory, [observation(200, 3)])
    query, cond = torch.randn(1, 2, D).cuda(), torch.randn(1, D).cuda()
    q_rot = L.rotary3d(torch.rand(1, 2, 3).cuda(), D)
    everything = stack(query, None, cond, q_rot, None, kv_caches=memory.layers)[0]
    memory.selected_pages = 16
    assert float((stack(query, None, cond, q_rot, None, kv_caches=memory.layers)[0] - everything).abs().max()) <= (STACK if dtype is torch.float32 else 0.05)
    memory.selected_pages = 3
    few = stack(query, None, cond, q_rot, None, kv_caches=memory.layers)[0]
    assert bool(torch.isfinite(few).all()) and not torch.equal(few, everything)


def test_memory_has_no_backward():
    stack = make_stack(3)
    memory = P.ContextMemory(2, 1, 16, H, 15, 16)
    with torch.no_grad():
        remember(stack, memory, [observation(20, 3)])
    with pytest.raises(RuntimeError, match="no backward"):
        stack(torch.randn(1, 2, D).cuda(), None, torch.randn(1, D).cuda(), None, None, kv_caches=memory.layers)
    with torch.no_grad(), pytest.raises(ValueError, match="weights"):
        stack(torch.randn(1, 2, D).cuda(), None, torch.randn(1, D).cuda(), None, None, kv_caches=memory.layers, need_weights=True)


@pytest.mark.parametrize("on", [False, True], ids=["composite", "fused"])
@torch.no_grad()
def test_model_with_a_memory(fused, on):
    """One observation in the memory is that observation; a second one adds to it; graph sampling leaves such a call alone."""
    torch.manual_seed(0)
    cfg = DiffuserActorConfig(data_type="mesh", feature_dim=16, diffusion_timesteps=3)
    bounds = torch.tensor([[-1.0, -1, -1], [1, 1, 1]])
    model = DiffuserActor(cfg, bounds).cuda().eval()
    fused(on)
    g = torch.Generator().manual_seed(3)

    def inputs():
        feats, verts = torch.randn(2, 300, 16, generator=g), torch.rand(2, 300, 3, generator=g) * 1.8 - 0.9
        valid = torch.rand(2, 300, generator=g) > 0.3
        pose = torch.cat([torch.rand(2, 3, 2, 3, generator=g), torch.nn.functional.normalize(torch.randn(2, 3, 2, 4, generator=g), dim=-1),
                          torch.ones(2, 3, 2, 1)], -1)
        return [None, None, None, None, None, feats.cuda(), verts.cuda(), valid.cuda(), None, pose.cuda()]

    one, two = inputs(), inputs()

    def run(args, memory=None):
        torch.manual_seed(11)
        return model(*args, run_inference=True, context_memory=memory)[0]

    memory = model.new_context_memory(2, 64, 32)
    plain, kept = run(one), run(one, memory)
    assert memory.held == tuple(one[7].sum(1).tolist())
    # three denoising steps of a random network over two evaluations of its attention: positions in metres
    assert float((plain - kept)[..., :3].abs().max()) <= 5e-3
    more = run(two, memory)
    assert memory.held == tuple((one[7].sum(1) + two[7].sum(1)).tolist()) and bool(torch.isfinite(more).all())
    assert not torch.equal(more, run(two))
    memory.release(0), memory.release(1)
    model.enable_graph_sampling()
    graphed, again = run(one), run(one, memory)
    assert float((graphed - again)[..., :3].abs().max()) <= 5e-3 and len(model._graph_sampler._graphs) == 1
    with pytest.raises(ValueError, match="contexts"):
        run(one, model.new_context_memory(3, 64, 32))


@pytest.mark.parametrize("case", ["width", "type", "positions", "rotary", "pool", "gradient"])
def test_a_refused_append_leaves_the_memory_as_it_was(case):
    memory = P.ContextMemory(2, 2, 4, 2, 16, 16)
    first = torch.randn(5, 32, generator=torch.Generator().manual_seed(1)).cuda()
    memory.append([3, 2], [(first, first)] * 2)
    state = lambda: [memory.pages_of.table.clone(), memory.pages_of.lengths.clone()] + [  # noqa: E731
        t.clone() for layer in memory.layers for t in (layer.pages.keys, layer.pages.values, layer.pages.key_min, layer.pages.key_max)]
    before, held, free = state(), memory.held, memory.pages_of.free_pages
    good, counts, positions, rotary = torch.ones(20, 32).cuda(), [17, 3], None, None
    bad = good
    if case == "width":
        bad = torch.ones(20, 30).cuda()
    elif case == "type":
        bad = good.half()
    elif case == "positions":
        positions = torch.zeros(19, 1).cuda()
    elif case == "rotary":
        positions, rotary = torch.zeros(20, 3).cuda(), 16
    elif case == "pool":
        counts, good, bad = [60, 20], torch.ones(80, 32).cuda(), torch.ones(80, 32).cuda()
    else:
        bad = good.clone().requires_grad_()
    with pytest.raises((ValueError, RuntimeError)):
        memory.append(counts, [(good, good), (bad, bad)], positions, rotary)
    assert memory.held == held and memory.pages_of.free_pages == free
    for x, y in zip(state(), before):
        assert torch.equal(x, y)


def test_the_page_table_is_not_changed_in_a_capture():
    t = P.PageTable(2, 6, 16)
    t.extend([17, 1])
    x = torch.zeros(64, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        x += 1
        for call in (lambda: t.extend([1, 1]), lambda: t.release(0)):
            with pytest.raises(RuntimeError, match="outside a captured graph"):
                call()
    g.replay()
    torch.cuda.synchronize()
    assert t.held == (17, 1) and t.lengths.tolist() == [17, 1] and t.free_pages == 3 and float(x.sum()) == 64.0
