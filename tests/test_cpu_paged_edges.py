"""What the paged context operators and their bookkeeping do at the edges, where no GPU is needed."""
import ctypes as C

import pytest
import torch

from nvblox_mindmap_amd import _lib
from nvblox_mindmap_amd.diffuser_actor import paged_context as P


def pages():
    low, high = torch.zeros(4, 2, 32), torch.zeros(4, 2, 32)
    return P.ContextPages(torch.zeros(4, 2, 16, 32), torch.zeros(4, 2, 32, 16), low, high, 20)


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.fixture
def host_only(monkeypatch):
    """The operators' checks on CPU tensors: the calls that pass them are collected instead of launched."""
    calls = []
    monkeypatch.setattr(P, "_check_device", lambda *args: None)
    monkeypatch.setattr(P, "_launch", lambda *args: calls.append(args))
    return calls


@pytest.mark.parametrize("count", [2 ** 30, 2 ** 31 - 1])
def test_selection_refuses_counts_that_its_index_would_pass(host_only, count):
    """The fill behind a row's last page steps on from an index below count: it has to stay in 32 bits."""
    fake = C.c_void_p(4096)
    rc = _lib.lib().mmf_paged_select(fake, fake, fake, 0, fake, fake, 1, 1, 1, 1, 20, 100, 4, 16, count, fake, fake, 1 << 30, None)
    assert rc != 0 and "count is below 2^30" in _lib.last_error()
    with pytest.raises(ValueError, match="below 2"):
        P.select_pages(torch.zeros(1, 1, 40), pages(), ints(1, 2), ints(1), 2, count)
    assert not host_only


def test_an_append_that_the_library_refuses_leaves_the_memory_as_it_was(host_only, monkeypatch):
    m = P.ContextMemory(2, 3, 12, 2, 16, 16, device="cpu")
    rows = lambda n: [(torch.zeros(n, 32), torch.zeros(n, 32))] * 2  # noqa: E731
    m.append([17, 0, 3], rows(20))
    t = m.pages_of
    before = (t.table.clone(), t.lengths.clone(), m.held, list(t._free), [list(p) for p in t._pages])

    def refused(*args):
        raise RuntimeError("mmf_paged_append: too many tokens or heads for one call")

    with monkeypatch.context() as patch:
        patch.setattr(P, "_launch", refused)
        with pytest.raises(RuntimeError, match="too many"):
            m.append([16, 40, 1], rows(57))
    assert torch.equal(t.table, before[0]) and torch.equal(t.lengths, before[1])
    assert (m.held, t._free, t._pages) == before[2:]
    m.append([16, 40, 1], rows(57))
    assert m.held == (33, 40, 4) and len(host_only) == 4


@pytest.mark.parametrize("autocast", [torch.bfloat16, torch.float16, None], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_an_observation_is_remembered_under_autocast(host_only, autocast, dtype):
    """Projections of either half type go into pages of any type."""
    from nvblox_mindmap_amd.diffuser_actor import DiffuserActor, DiffuserActorConfig

    model = DiffuserActor(DiffuserActorConfig(data_type="mesh", feature_dim=8), torch.tensor([[-1.0, -1, -1], [1, 1, 1]]))
    memory = model.new_context_memory(2, 8, 16, dtype, device="cpu")
    enc = {"context_feats": torch.randn(2, 9, 120), "context_pos": torch.rand(2, 9, 3), "context_mask": torch.rand(2, 9) < 0.7}
    with torch.no_grad(), torch.autocast("cpu", autocast or torch.bfloat16, enabled=autocast is not None):
        model.prediction_head.extend_memory(memory, enc)
    assert memory.held == tuple(enc["context_mask"].sum(1).tolist()) and len(host_only) == 2


@pytest.mark.parametrize("base", [float("inf"), float("nan"), -1.0])
def test_the_c_append_refuses_a_rotary_base_without_angles(base):
    fake = C.c_void_p(4096)
    rc = _lib.lib().mmf_paged_append(fake, 40, fake, 40, 0, 3, fake, 1, 20, base, fake, fake, fake, 1, 2, 16, 2, 20, 4, 0, fake, fake, fake, fake, None)
    assert rc != 0 and "positive, finite base" in _lib.last_error()


@pytest.mark.parametrize("entry,args", [("append", (0, 1, 2, 3)), ("attention", (0, 1, 2)), ("select", (0, 1, 2))])
def test_the_c_entries_refuse_unaligned_pools_and_workspaces(entry, args):
    fake, odd = C.c_void_p(4096), C.c_void_p(4104)
    for bad in args:
        p = [odd if i == bad else fake for i in range(4)]
        if entry == "append":
            rc = _lib.lib().mmf_paged_append(fake, 40, fake, 40, 0, 3, fake, 1, 20, 100.0, fake, fake, fake, 1, 2, 16, 2, 20, 4, 0, *p, None)
        elif entry == "attention":
            rc = _lib.lib().mmf_paged_attention(fake, p[0], p[1], 0, fake, fake, None, 0, 2, 1, 2, 1, 20, 100, 4, 256, 1.0, fake, p[2], 1 << 40, None)
        else:
            rc = _lib.lib().mmf_paged_select(fake, p[0], p[1], 0, fake, fake, 2, 1, 2, 1, 20, 100, 4, 16, 3, fake, p[2], 1 << 30, None)
        assert rc != 0 and "aligned to 16 bytes" in _lib.last_error()
