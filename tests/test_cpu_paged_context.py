"""Refusals of the paged context operators, and the sizes they answer without a GPU."""
import ctypes as C

import pytest
import torch

from nvblox_mindmap_amd import _lib
from nvblox_mindmap_amd.diffuser_actor import paged_context as P


def pages(**change):
    keys, values = torch.zeros(4, 2, 16, 32), torch.zeros(4, 2, 32, 16)
    low, high = torch.zeros(4, 2, 32), torch.zeros(4, 2, 32)
    d = dict(keys=keys, values=values, key_min=low, key_max=high, head_dim=20)
    d.update(change)
    return P.ContextPages(**d)


def test_head_width_agrees_with_the_library():
    L = _lib.lib()
    for hd in range(1, 257):
        assert P.head_width(hd) == L.mmf_paged_width(hd) >= hd
    assert L.mmf_paged_width(0) == 0 and L.mmf_paged_width(257) == 0 and L.mmf_paged_width(-1) == 0
    for hd in (0, 257):
        with pytest.raises(ValueError):
            P.head_width(hd)


def test_no_cpu_fallback():
    t = torch.zeros(1, 2, dtype=torch.int32)
    one = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        P.context_attention(torch.zeros(1, 1, 40), pages(), t, one, 2)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        P.select_pages(torch.zeros(1, 1, 40), pages(), t, one, 2, 1)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        P.append_context(pages(), torch.zeros(1, 40), torch.zeros(1, 40), torch.zeros(2, dtype=torch.int32), one, t)


@pytest.mark.parametrize("change,match", [
    (dict(keys=torch.zeros(4, 2, 24, 32)), "page_size"),
    (dict(head_dim=33), "head_dim"),
    (dict(head_dim=300), "head_dim"),
    (dict(values=torch.zeros(4, 2, 16, 32)), "values"),
    (dict(values=torch.zeros(4, 2, 32, 16, dtype=torch.float16)), "alike"),
    (dict(keys=torch.zeros(4, 2, 16, 32, dtype=torch.float64)), "float32, float16 or bfloat16"),
    (dict(keys=torch.zeros(4, 2, 32, 16).transpose(2, 3)), "contiguous"),
    (dict(key_min=None), "key_min"),
    (dict(key_max=torch.zeros(4, 2, 31)), "key_min"),
    (dict(key_max=torch.zeros(4, 2, 32, dtype=torch.float16)), "key_min"),
])
def test_pages_are_checked(change, match):
    with pytest.raises(ValueError, match=match):
        P._check_pages(pages(**change), True)


def test_allocation_is_checked():
    for bad in (dict(page_size=48), dict(dtype=torch.int8), dict(head_dim=0), dict(num_pages=0), dict(kv_heads=0)):
        args = dict(num_pages=2, kv_heads=2, head_dim=8, page_size=16, dtype=torch.float16, device="cpu")
        args.update(bad)
        with pytest.raises(ValueError):
            P.allocate_pages(**args)
    c = P.allocate_pages(3, 2, 15, 32, torch.bfloat16, "cpu")
    assert c.keys.shape == (3, 2, 32, 16) and c.values.shape == (3, 2, 16, 32) and c.key_min.shape == (3, 2, 16) and c.page_size == 32


def call_append(**change):
    """The C entry with addresses that are never read: every case below is refused before a launch."""
    fake = C.c_void_p(4096)
    d = dict(k=fake, ks=40, v=fake, vs=40, in_type=0, tokens=3, positions=fake, axes=1, rotary=20, base=10000.0, offsets=fake, starts=fake, table=fake, B=1,
             slots=2, page=16, heads=2, hd=20, num=4, type=0, keys=fake, values=fake, kmin=fake, kmax=fake, stream=None)
    d.update(change)
    return _lib.lib().mmf_paged_append(*d.values())


@pytest.mark.parametrize("change", [dict(page=24), dict(page=8), dict(page=512), dict(hd=0), dict(hd=257), dict(type=3), dict(type=-1), dict(in_type=1),
                                    dict(B=0), dict(slots=0), dict(slots=2 ** 28), dict(heads=0), dict(num=0), dict(tokens=-1), dict(tokens=2 ** 31),
                                    dict(axes=0), dict(axes=5), dict(rotary=21), dict(rotary=22), dict(rotary=-2), dict(base=0.0), dict(positions=None), dict(k=None), dict(keys=None),
                                    dict(kmin=None), dict(table=None), dict(ks=-1), dict(vs=2 ** 23), dict(heads=2 ** 22, hd=256, rotary=0),
                                    dict(tokens=2 ** 31 - 1, B=2 ** 28)])
def test_append_refuses(change):
    assert call_append(**change) != 0 and "mmf_paged_append" in _lib.last_error()


def call_attention(**change):
    fake = C.c_void_p(4096)
    d = dict(q=fake, keys=fake, values=fake, type=0, table=fake, lengths=fake, selected=None, count=0, B=2, T=1, heads=2, group=1, hd=20, slots=100, num=4,
             page=256, scale=1.0, out=fake, work=fake, bytes=1 << 40, stream=None)
    d.update(change)
    return _lib.lib().mmf_paged_attention(*d.values())


@pytest.mark.parametrize("change", [dict(page=17), dict(hd=300), dict(type=7), dict(B=0), dict(T=0), dict(group=0), dict(slots=0), dict(slots=2 ** 24), dict(num=0),
                                    dict(q=None), dict(lengths=None), dict(out=None), dict(bytes=0), dict(work=None),
                                    dict(selected=C.c_void_p(4096), count=0), dict(T=2 ** 25),
                                    dict(selected=C.c_void_p(4096), count=4, B=2 ** 15, T=2 ** 10), dict(heads=2 ** 20, B=2 ** 6, slots=4, page=16)])
def test_attention_refuses(change):
    assert call_attention(**change) != 0 and "mmf_paged_attention" in _lib.last_error()


@pytest.mark.parametrize("change", [dict(count=0), dict(T=0), dict(bytes=8), dict(work=None), dict(type=3), dict(page=0), dict(kmin=None), dict(group=0), dict(B=2 ** 14, T=2 ** 10, bytes=1 << 50)])
def test_selection_refuses(change):
    fake = C.c_void_p(4096)
    d = dict(q=fake, kmin=fake, kmax=fake, type=0, table=fake, lengths=fake, B=2, T=1, heads=2, group=1, hd=20, slots=100, num=4, page=16, count=3, out=fake,
             work=fake, bytes=1 << 30, stream=None)
    d.update(change)
    assert _lib.lib().mmf_paged_select(*d.values()) != 0 and "mmf_paged_select" in _lib.last_error()


# ---- refusals of the operators' arguments, which are found on the host: on CPU tensors with the device check taken out ----
@pytest.fixture
def host_only(monkeypatch):
    def reached(*args):
        raise AssertionError("a call that has to be refused reached the library")

    monkeypatch.setattr(P, "_check_device", lambda *args: None)
    monkeypatch.setattr(P, "_launch", reached)


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


LONG = 2 ** 31


@pytest.mark.parametrize("change,match", [
    (dict(k=torch.zeros(3, 41)), "k and v"),
    (dict(k=torch.zeros(3, 40).half()), "both alike"),
    (dict(k=torch.zeros(3, 40).half(), v=torch.zeros(3, 40).half()), "float32"),
    (dict(v=torch.zeros(2, 40)), "k and v"),
    (dict(starts=torch.zeros(1, dtype=torch.int64)), "starts"),
    (dict(offsets=ints(1)), "offsets"),
    (dict(offsets=ints(4)[::2]), "offsets"),
    (dict(table=ints(2)), "table"),
    (dict(table=ints(2, 2)), "starts"),
    (dict(positions=torch.zeros(2, 1)), "positions"),
    (dict(positions=torch.zeros(3, 5)), "positions"),
    (dict(positions=torch.zeros(3, 1, dtype=torch.float64)), "positions"),
    (dict(positions=torch.zeros(3, 1), rotary_dim=30), "rotary_dim"),
    (dict(positions=torch.zeros(3, 1), rotary_dim=0), "rotary_dim"),
    (dict(positions=torch.zeros(3, 3), rotary_dim=20), "rotary_dim"),
    (dict(positions=torch.zeros(3, 1), rotary_base=0.0), "rotary_base"),
    (dict(positions=torch.zeros(3, 1), rotary_base=float("inf")), "rotary_base"),
    (dict(positions=torch.zeros(3, 1), rotary_base=float("nan")), "rotary_base"),
    (dict(rotary_dim=20), "without positions"),
    (dict(k=torch.zeros(1, 40).expand(LONG, 40), v=torch.zeros(1, 40).expand(LONG, 40)), "below 2"),
    (dict(table=torch.empty(1, LONG, dtype=torch.int32)), "below 2"),
])
def test_append_context_refuses(host_only, change, match):
    d = dict(k=torch.zeros(3, 40), v=torch.zeros(3, 40), offsets=ints(2), starts=ints(1), table=ints(1, 2))
    d.update(change)
    with pytest.raises(ValueError, match=match):
        P.append_context(pages(), **d)


QUERY = [
    (dict(heads=3), "multiple"),
    (dict(heads=0), "multiple"),
    (dict(q=torch.zeros(1, 1, 39)), "q "),
    (dict(q=torch.zeros(1, 40)), "q "),
    (dict(q=torch.zeros(1, 1, 40).half()), "the pages are"),
    (dict(table=ints(2, 2)), "contexts"),
    (dict(lengths=ints(2)), "contexts"),
    (dict(lengths=torch.zeros(1)), "lengths"),
    (dict(table=ints(1, 4)[:, ::2]), "table"),
    (dict(q=torch.zeros(1, 1, 40).expand(1, LONG, 40)), "below 2"),
    (dict(table=torch.empty(1, LONG, dtype=torch.int32)), "below 2"),
]


def query(**change):
    d = dict(q=torch.zeros(1, 1, 40), context=pages(), table=ints(1, 2), lengths=ints(1), heads=2)
    d.update(change)
    return d


@pytest.mark.parametrize("change,match", QUERY + [
    (dict(pages=ints(1, 1, 2)), "pages"),
    (dict(pages=ints(1, 2, 2, 3)), "pages"),
    (dict(pages=torch.zeros(1, 1, 2, 3, dtype=torch.int64)), "pages"),
])
def test_context_attention_refuses(host_only, change, match):
    with pytest.raises(ValueError, match=match):
        P.context_attention(**query(**change))


@pytest.mark.parametrize("change,match", QUERY + [(dict(count=0), "count"), (dict(count=-1), "count"), (dict(count=LONG), "below 2"),
                                                  (dict(count=2 ** 32 + 5), "below 2"), (dict(context=pages(key_min=None)), "key_min")])
def test_select_pages_refuses(host_only, change, match):
    with pytest.raises(ValueError, match=match):
        P.select_pages(**{**query(count=2), **query(**change)} if "count" in change else {**query(**change), "count": 2})


def test_workspace_sizes():
    L = _lib.lib()
    assert L.mmf_paged_select_workspace_bytes(2, 3, 4, 5) >= 8 * 120
    assert L.mmf_paged_attention_workspace_bytes(1, 1, 1, 1, 16, 100, 0) == 0  # one split: no partial results
    assert L.mmf_paged_attention_workspace_bytes(1, 1, 8, 4, 128, 1 << 20, 0) > 0
    assert L.mmf_paged_attention_workspace_bytes(0, 1, 8, 4, 128, 1 << 20, 0) == 0


# ---- the page table -------------------------------------------------------------------------------------------------------------------
def test_page_table_hands_out_each_page_once():
    t = P.PageTable(3, 10, 16, slots=6, device="cpu")
    offsets, starts = t.extend([17, 0, 16])
    assert offsets.tolist() == [0, 17, 17, 33] and starts.tolist() == [0, 0, 0] and offsets.dtype == starts.dtype == torch.int32
    assert t.held == (17, 0, 16) and t.lengths.tolist() == [17, 0, 16] and t.free_pages == 7
    offsets, starts = t.extend([15, 1, 1])  # context 0 fills its second page
    assert starts.tolist() == [17, 0, 16] and t.free_pages == 5
    used = [p for p in t.table.flatten().tolist() if p >= 0]
    assert sorted(used) == sorted(set(used)) and len(used) == 5 and (t.table[0] >= 0).sum() == 2
    before = (t.table.clone(), t.held, t.free_pages)
    with pytest.raises(RuntimeError, match="free"):
        t.extend([0, 80, 16])
    with pytest.raises(RuntimeError, match="would pass"):
        t.extend([65, 0, 0])
    for bad in ([1, 2], [1, -1, 0]):
        with pytest.raises(ValueError):
            t.extend(bad)
    assert torch.equal(t.table, before[0]) and t.held == before[1] and t.free_pages == before[2]
    t.release(0)
    assert t.free_pages == 7 and t.held == (0, 1, 17) and t.table[0].tolist() == [-1] * 6 and t.lengths.tolist() == [0, 1, 17]
    t.extend([96, 0, 0])
    used = [p for p in t.table.flatten().tolist() if p >= 0]
    assert len(used) == len(set(used)) == 9


def test_page_table_made_in_inference_mode_is_used_outside():
    with torch.inference_mode():
        t = P.PageTable(2, 6, 16, device="cpu")
    t.extend([17, 1])
    with torch.inference_mode():
        t.extend([0, 16])
    t.release(0)
    assert t.held == (0, 17) and t.lengths.tolist() == [0, 17] and t.free_pages == 4


def test_page_table_keeps_its_books_where_the_device_fails(monkeypatch):
    t = P.PageTable(2, 6, 16, device="cpu")
    t.extend([17, 1])
    table, held, free, pages_ = t.table, t.held, t.free_pages, [list(p) for p in t._pages]

    class Broken:
        device, is_cuda = table.device, False

        def __setitem__(self, at, value):
            raise RuntimeError("no memory")

        def __getitem__(self, at):
            raise RuntimeError("no memory")

    monkeypatch.setattr(t, "table", Broken())
    for call in (lambda: t.extend([16, 16]), lambda: t.release(0)):
        with pytest.raises(RuntimeError, match="no memory"):
            call()
    monkeypatch.setattr(t, "table", table)
    assert t.held == held and t.free_pages == free and t._pages == pages_ and t.lengths.tolist() == [17, 1]


def test_memory_is_checked():
    with pytest.raises(ValueError):
        P.ContextMemory(0, 1, 4, 2, 16, 16, device="cpu")
    with pytest.raises(ValueError):
        P.ContextMemory(1, 1, 4, 2, 16, 16, selected_pages=0, device="cpu")
    with pytest.raises(ValueError):
        P.PageTable(1, 4, 17, device="cpu")
    m = P.ContextMemory(2, 2, 4, 2, 16, 16, device="cpu")
    k = torch.zeros(3, 32)
    with pytest.raises(ValueError, match="2 layers"):
        m.append([1, 2], [(k, k)])
    with pytest.raises(ValueError, match="of 4 tokens"):
        m.append([1, 3], [(k, k), (k, k)])
    assert m.held == (0, 0)


def test_a_refused_append_leaves_the_memory_as_it_was():
    m = P.ContextMemory(2, 2, 4, 2, 16, 16, device="cpu")
    k = torch.zeros(3, 32)
    before = m.pages_of.table.clone()
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        m.append([1, 2], [(k, k), (k, k)])
    assert m.held == (0, 0) and m.pages_of.free_pages == 4
    assert torch.equal(m.pages_of.table, before) and m.pages_of.lengths.tolist() == [0, 0]


def test_model_refuses_a_memory_where_it_has_no_meaning():
    from nvblox_mindmap_amd.diffuser_actor import DiffuserActor, DiffuserActorConfig

    cfg = DiffuserActorConfig(data_type="mesh", feature_dim=8, relative_action=True)
    model = DiffuserActor(cfg, torch.tensor([[-1.0, -1, -1], [1, 1, 1]]))
    memory = model.new_context_memory(1, 4, 16, device="cpu")
    assert len(memory.layers) == 2 and memory.layers[0].pages.head_dim == 15
    args = [None] * 10
    args[9] = torch.zeros(1, 3, 2, 8)
    with pytest.raises(ValueError, match="inference"):
        model(*args, context_memory=memory)
    with torch.no_grad(), pytest.raises(ValueError, match="relative_action"):
        model(*args, run_inference=True, context_memory=memory)
