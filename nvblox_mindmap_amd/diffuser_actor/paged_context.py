"""Keys and values of growing contexts in pages, and the attention over them (libmmfusion: mmf_paged_append, mmf_paged_attention,
mmf_paged_select; csrc/mmf_kernels_paged.hip).

The policy's cross-attention (mindmap/diffuser_actor/diffusion_head.py) reads one observation's context, projected anew for every
inference and padded to one length per batch.  Here a context grows: its tokens' keys (rotated by their position on the way in) and
values are kept in pages of ``page_size`` tokens, so contexts of unlike length share one pool without padding, what was seen before
is not projected again, and a long context can be attended to through its few relevant pages.

``ContextPages`` names the buffers of one layer, ``append_context`` / ``context_attention`` / ``select_pages`` are the operators over
them (float32, float16, bfloat16; no autograd; nothing synchronises, all lengths are read on the device, so calls can be captured into
a graph and replayed with other lengths).  ``PageTable`` hands out a pool's pages to contexts, ``ContextMemory`` puts the table and the
pages of a stack's layers together: what ``DiffuserActor`` keeps of earlier observations (``new_context_memory``)."""
import functools
import math
from typing import List, NamedTuple, Optional, Sequence, Tuple

import torch
from torch.autograd import forward_ad

from .. import _lib

WIDTHS = (16, 32, 64, 96, 128, 256)  # head sizes the pages are laid out for; a head is padded to the next (mmf_paged_width)
PAGE_SIZES = (16, 32, 64, 128, 256)
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def head_width(head_dim: int) -> int:
    for w in WIDTHS:
        if 1 <= head_dim <= w:
            return w
    raise ValueError(f"head_dim {head_dim}: 1 to {WIDTHS[-1]} are supported")


class ContextPages(NamedTuple):
    """The pages of one attention layer.
      keys    [num_pages, kv_heads, page_size, W]   a token's channels side by side
      values  [num_pages, kv_heads, W, page_size]   a channel's tokens side by side
      key_min, key_max [num_pages, kv_heads, W]     smallest / largest stored key of a page per channel (None: no selection, no append)
    W = head_width(head_dim); channels behind head_dim are zero."""

    keys: torch.Tensor
    values: torch.Tensor
    key_min: Optional[torch.Tensor]
    key_max: Optional[torch.Tensor]
    head_dim: int

    @property
    def page_size(self) -> int:
        return self.keys.shape[2]


def allocate_pages(num_pages: int, kv_heads: int, head_dim: int, page_size: int = 64, dtype: torch.dtype = torch.float32,
                   device="cuda") -> ContextPages:
    """Empty pages (zeroed: the padding channels have to be)."""
    if dtype not in _TYPES:
        raise ValueError(f"pages are float32, float16 or bfloat16, not {dtype}")
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size {page_size}: one of {PAGE_SIZES}")
    if num_pages < 1 or kv_heads < 1:
        raise ValueError("num_pages and kv_heads have to be positive")
    w = head_width(head_dim)
    zeros = lambda *shape: torch.zeros(shape, dtype=dtype, device=device)  # noqa: E731
    return ContextPages(zeros(num_pages, kv_heads, page_size, w), zeros(num_pages, kv_heads, w, page_size), zeros(num_pages, kv_heads, w),
                        zeros(num_pages, kv_heads, w), head_dim)


# ---- checks: one expression on the way to the kernel (a call's host time is a good part of a small call), the reason only where it fails ----
def _pages_ok(c: ContextPages, summary: bool) -> bool:
    k, v, lo, hi, hd = c
    shape = k.shape
    if len(shape) != 4:
        return False
    n, h, p, w = shape
    dtype, index = k.dtype, k.get_device()
    ok = (dtype in _TYPES and v.dtype is dtype and p in PAGE_SIZES and n > 0 and h > 0 and 1 <= hd <= 256 and w == _WIDTH_OF[hd]
          and v.shape == (n, h, w, p) and k.is_contiguous() and v.is_contiguous() and v.get_device() == index
          and not (k.data_ptr() | v.data_ptr()) & 15)
    if ok and summary:
        shape = (n, h, w)
        ok = (lo is not None and hi is not None and lo.shape == shape and hi.shape == shape and lo.dtype is dtype and hi.dtype is dtype
              and lo.is_contiguous() and hi.is_contiguous() and lo.get_device() == index and hi.get_device() == index
              and not (lo.data_ptr() | hi.data_ptr()) & 15)
    return ok


_WIDTH_OF = (0,) + tuple(next(w for w in WIDTHS if w >= d) for d in range(1, WIDTHS[-1] + 1))


def _check(cond: bool, what: str) -> None:
    if not cond:
        raise ValueError(what)


_LONG = 31  # sizes of a call, or-ed together and shifted: the library takes 32-bit sizes, and a longer one would reach it cut off


def _too_long(*sizes: int) -> ValueError:
    return ValueError(f"sizes of a call are below 2^31: got {max(sizes)}")


def _check_pages(c: ContextPages, summary: bool) -> None:
    if _pages_ok(c, summary):
        return
    k, v = c.keys, c.values
    _check(k.dim() == 4 and v.dim() == 4, "keys [pages, kv_heads, page_size, W] and values [pages, kv_heads, W, page_size]")
    n, h, p, w = k.shape
    _check(k.dtype in _TYPES and v.dtype == k.dtype, f"pages are float32, float16 or bfloat16, all alike: got {k.dtype}, {v.dtype}")
    _check(p in PAGE_SIZES, f"page_size {p}: one of {PAGE_SIZES}")
    _check(w == head_width(c.head_dim), f"head_dim {c.head_dim} has pages of {head_width(c.head_dim)} channels, not {w}")
    _check(v.shape == (n, h, w, p), f"values {tuple(v.shape)} do not go with keys {tuple(k.shape)}")
    _check(n > 0 and h > 0, "no pages")
    _check(v.device == k.device, "pages on one device")
    _check(not summary or (c.key_min is not None and c.key_max is not None), "pages without key_min / key_max")
    for s in (c.key_min, c.key_max) if summary else ():
        _check(s.shape == (n, h, w) and s.dtype == k.dtype and s.device == k.device, "key_min / key_max [pages, kv_heads, W] of the pages' type, on their device")
    raise ValueError("pages are contiguous and 16-byte aligned")


def _ints_ok(t: torch.Tensor, dim: int, index: int) -> bool:
    return t.dtype is torch.int32 and t.dim() == dim and t.get_device() == index and t.is_contiguous()


def _check_ints(keys: torch.Tensor, **ts: Tuple[torch.Tensor, int]) -> None:
    for name, (t, dim) in ts.items():
        _check(_ints_ok(t, dim, keys.get_device()), f"{name}: a contiguous int32 tensor of {dim} dimension(s) on {keys.device}")


def _no_backward() -> RuntimeError:
    return RuntimeError("paged contexts have no backward pass: call them under torch.no_grad(), or detach the inputs")


def _check_device(index: int, keys: torch.Tensor, values: torch.Tensor, *ts: Optional[torch.Tensor]) -> None:
    """The inputs ``ts`` on the pages' device; no derivative in them or in the pages (whose devices _pages_ok compares)."""
    if index < 0:
        raise RuntimeError("paged contexts live on an MI355X (no CPU fallback)")
    grad = torch.is_grad_enabled()
    for t in ts:
        if t is not None:
            if t.get_device() != index:
                raise ValueError(f"all tensors on cuda:{index}: got one on {t.device}")
            if grad and t.requires_grad:
                raise _no_backward()
    if grad and (keys.requires_grad or values.requires_grad):
        raise _no_backward()
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in (keys, values, *ts)):
        raise _no_backward()


def _launch(index: int, entry, what: str, *args) -> None:
    """entry(*args, stream) on the current stream of device `index`, which is made current for the call where it is not."""
    current = torch._C._cuda_getDevice()
    if current == index:
        rc = entry(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = entry(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc, what)


@functools.lru_cache(maxsize=512)
def _attention_bytes(B, T, H, G, hd, capacity, selected) -> int:
    return int(_lib.lib().mmf_paged_attention_workspace_bytes(B, T, H, G, hd, capacity, selected))


@functools.lru_cache(maxsize=512)
def _select_bytes(B, T, H, slots) -> int:
    return int(_lib.lib().mmf_paged_select_workspace_bytes(B, T, H, slots))


def _check_rows(context: ContextPages, k: torch.Tensor, v: torch.Tensor, positions: Optional[torch.Tensor], rotary_dim: Optional[int],
                rotary_base: float) -> Tuple[int, int, int, int]:
    """What ``append_context`` asks of the pages and the rows.  -> (rows, axes, rotated channels, address of the positions)"""
    keys, hd = context.keys, context.head_dim
    _check_device(keys.get_device(), keys, context.values, k, v, positions)
    if not _pages_ok(context, True):
        _check_pages(context, True)
    row = keys.shape[1] * hd
    shape = k.shape
    if not (len(shape) == 2 and shape[1] == row and v.shape == shape):
        raise ValueError(f"k and v [n, {row}]: got {tuple(k.shape)}, {tuple(v.shape)}")
    dtype, n = k.dtype, shape[0]
    if not (v.dtype is dtype and (dtype is keys.dtype or dtype is torch.float32)):
        raise ValueError(f"k and v are {keys.dtype} or float32, both alike: got {k.dtype}, {v.dtype}")
    if positions is None:
        if rotary_dim is not None:
            raise ValueError("rotary_dim without positions")
        return n, 1, 0, 0
    shape = positions.shape
    if not (len(shape) == 2 and shape[0] == n and 1 <= shape[1] <= 4 and positions.dtype is torch.float32 and positions.is_contiguous()):
        raise ValueError(f"positions [{n}, axes] float32, contiguous, 1 to 4 axes")
    axes, rotary = shape[1], row if rotary_dim is None else int(rotary_dim)
    if not (rotary > 0 and rotary % (2 * axes) == 0 and (rotary <= hd or rotary == row)):
        raise ValueError(f"rotary_dim {rotary}: a multiple of {2 * axes}, at most head_dim {hd} or the whole row {row}")
    if not 0 < rotary_base < math.inf:
        raise ValueError("rotary_base has to be positive and finite")
    return n, axes, rotary, positions.data_ptr()


def append_context(context: ContextPages, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor, starts: torch.Tensor, table: torch.Tensor,
                   positions: Optional[torch.Tensor] = None, rotary_dim: Optional[int] = None, rotary_base: float = 10000.0) -> None:
    """Rows ``offsets[b] : offsets[b + 1]`` of k and v [n, kv_heads * head_dim] (the pages' type or float32; rows may be strided) become
    tokens ``starts[b]``, ``starts[b] + 1``, ... of context b, in the pages ``table[b]`` [contexts, slots] names; rows behind
    ``offsets[-1]``, and tokens whose table entry is outside [0, num_pages) or behind the table, are not stored.

    With ``positions`` [n, axes] (float32, 1 to 4 axes) the keys are rotated on the way as ``layers.rotary3d`` / ``apply_rotary`` do (pairs
    of neighbouring channels, 2 i with 2 i + 1; a rotation of a head's halves is not offered):
    ``rotary_dim`` channels, each axis a share of them.  rotary_dim = kv_heads * head_dim (the default): one code over the whole row, the
    policy's; rotary_dim <= head_dim: the first channels of every head.  Angles are taken in 64 bits (far positions keep their fraction).

    A page gets tokens of one context in a call (two that append to one page in the same call leave it undefined); pages that are only
    read may be shared."""
    keys, values, low, high, hd = context
    n, axes, rotary, at = _check_rows(context, k, v, positions, rotary_dim, rotary_base)
    index = keys.get_device()
    if not (_ints_ok(table, 2, index) and _ints_ok(starts, 1, index) and _ints_ok(offsets, 1, index)):
        _check_ints(keys, table=(table, 2), starts=(starts, 1), offsets=(offsets, 1))
    n_pages, h, p, _ = keys.shape
    b, slots = table.shape
    if (n | b | slots) >> _LONG:
        raise _too_long(n, b, slots)
    if not (starts.numel() == b and offsets.numel() == b + 1):
        raise ValueError(f"{b} contexts have {b} starts and {b + 1} offsets")
    if n == 0 or b == 0 or slots == 0:
        return
    (k_stride, k_step), (v_stride, v_step) = k.stride(), v.stride()
    if k_step != 1 or k_stride >= 1 << 23:
        k, k_stride = k.contiguous(), h * hd
    if v_step != 1 or v_stride >= 1 << 23:
        v, v_stride = v.contiguous(), h * hd
    _launch(index, _lib.lib().mmf_paged_append, "mmf_paged_append", k.data_ptr(), k_stride, v.data_ptr(), v_stride, _TYPES[k.dtype], n, at, axes,
            rotary, rotary_base, offsets.data_ptr(), starts.data_ptr(), table.data_ptr(), b, slots, p, h, hd, n_pages, _TYPES[keys.dtype], keys.data_ptr(),
            values.data_ptr(), low.data_ptr(), high.data_ptr())


def _check_query(q: torch.Tensor, context: ContextPages, table: torch.Tensor, lengths: torch.Tensor, heads: int, summary: bool) -> Tuple[int, int, int]:
    """What the attention and the selection ask of pages, query and table.  -> (contexts, tokens, slots)"""
    keys = context.keys
    index = keys.get_device()
    _check_device(index, keys, context.values, q)
    if not _pages_ok(context, summary):
        _check_pages(context, summary)
    h = keys.shape[1]
    if not (heads > 0 and heads % h == 0):
        raise ValueError(f"heads {heads}: a multiple of the {h} key-value heads")
    shape, row = q.shape, heads * context.head_dim
    if not (len(shape) == 3 and shape[2] == row):
        raise ValueError(f"q [contexts, tokens, {row}]: got {tuple(shape)}")
    if q.dtype is not keys.dtype:
        raise ValueError(f"q is {q.dtype}, the pages are {keys.dtype}")
    if not (_ints_ok(table, 2, index) and _ints_ok(lengths, 1, index)):
        _check_ints(keys, table=(table, 2), lengths=(lengths, 1))
    b, t, _ = shape
    contexts, slots = table.shape
    if (b | t | row | slots) >> _LONG:
        raise _too_long(b, t, row, slots)
    if not contexts == b == lengths.numel():
        raise ValueError(f"{b} contexts: table {tuple(table.shape)}, lengths {tuple(lengths.shape)}")
    return b, t, slots


def context_attention(q: torch.Tensor, context: ContextPages, table: torch.Tensor, lengths: torch.Tensor, heads: int,
                      scale: Optional[float] = None, pages: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale q k^T) v per head over the first ``lengths[b]`` tokens of context b (scale: 1 / sqrt(head_dim) unless given); q
    [contexts, T, heads * head_dim] of the pages' type, rotated by the caller (``fused_ops.rotary_apply``, ``q_block``); query head i reads
    key-value head i // (heads / kv_heads).  ``pages`` [contexts, T, kv_heads, count] int32 (``select_pages``): over the tokens of these
    table slots only; an entry outside the table holds nothing, none may stand twice.  Zeros where there is no token.  -> [contexts, T, heads * head_dim].
    A pass over keys and values serves 32 query rows of a key-value head (T * heads / kv_heads; 16 where head_dim > 128): meant for few tokens."""
    b, t, slots = _check_query(q, context, table, lengths, heads, False)
    keys, values, _, _, hd = context
    index = keys.get_device()
    n_pages, h, p, _ = keys.shape
    count, chosen = 0, 0
    if pages is not None:
        if not _ints_ok(pages, 4, index):
            _check_ints(keys, pages=(pages, 4))
        count, chosen = pages.shape[3], pages.data_ptr()
        if count >> _LONG:
            raise _too_long(count)
        if pages.shape != (b, t, h, count):
            raise ValueError(f"pages [{b}, {t}, {h}, count]: got {tuple(pages.shape)}")
    if b == 0 or t == 0 or slots == 0 or (pages is not None and count == 0):
        return torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    if not q.is_contiguous():
        q = q.contiguous()
    out = torch.empty_like(q)
    need = _attention_bytes(b, t, h, heads // h, hd, (slots if pages is None else count) * p, int(pages is not None))
    # per call, from torch's caching allocator: safe inside a captured graph (its private pool) and across streams
    work = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    _launch(index, _lib.lib().mmf_paged_attention, "mmf_paged_attention", q.data_ptr(), keys.data_ptr(), values.data_ptr(), _TYPES[q.dtype],
            table.data_ptr(), lengths.data_ptr(), chosen, count, b, t, h, heads // h, hd, slots, n_pages, p, hd ** -0.5 if scale is None else scale,
            out.data_ptr(), work.data_ptr() if need else 0, need)
    return out


def select_pages(q: torch.Tensor, context: ContextPages, table: torch.Tensor, lengths: torch.Tensor, heads: int, count: int) -> torch.Tensor:
    """Table slots of the ``count`` pages that can hold the largest products with each query token, for every key-value head:
    [contexts, T, kv_heads, count] int32, ascending, filled up with -1 -- the ``pages`` of ``context_attention``.  A page's score is
    sum_c max(q_c, 0) key_max_c + min(q_c, 0) key_min_c, which no key of the page exceeds, the largest over the query heads that share the
    key-value head; taken in 64 bits, the lower slot first among equals.  Time and workspace (8 bytes a slot, token and key-value head) follow
    the table's width, whatever the lengths."""
    b, t, slots = _check_query(q, context, table, lengths, heads, True)
    keys, _, low, high, hd = context
    index = keys.get_device()
    if not count > 0:
        raise ValueError("count has to be positive")
    if count >> 30:
        raise ValueError(f"count is below 2^30: got {count}")
    n_pages, h, p, _ = keys.shape
    if b == 0 or t == 0 or slots == 0:
        return torch.full((b, t, h, count), -1, dtype=torch.int32, device=q.device)
    if not q.is_contiguous():
        q = q.contiguous()
    out = torch.empty((b, t, h, count), dtype=torch.int32, device=q.device)
    need = _select_bytes(b, t, h, slots)
    work = torch.empty(need, dtype=torch.uint8, device=q.device)
    _launch(index, _lib.lib().mmf_paged_select, "mmf_paged_select", q.data_ptr(), low.data_ptr(), high.data_ptr(), _TYPES[q.dtype],
            table.data_ptr(), lengths.data_ptr(), b, t, h, heads // h, hd, slots, n_pages, p, count, out.data_ptr(), work.data_ptr(), need)
    return out


class PageTable:
    """Which pages of a pool belong to which context: the bookkeeping on the host, ``table`` [contexts, slots] and ``lengths`` [contexts] int32
    on the device, changed in place (a captured graph reads the new ones).  A page belongs to one context.  ``slots``: the most pages of a
    context, all of the pool unless given -- give its share where many contexts share a pool and pages are selected (``select_pages``)."""

    def __init__(self, contexts: int, num_pages: int, page_size: int, slots: Optional[int] = None, device="cuda"):
        if contexts < 1 or num_pages < 1 or page_size not in PAGE_SIZES:
            raise ValueError(f"positive sizes, page_size one of {PAGE_SIZES}")
        self.page_size, self.num_pages = page_size, num_pages
        self.slots = num_pages if slots is None else int(slots)
        if self.slots < 1:
            raise ValueError("slots has to be positive")
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages: List[List[int]] = [[] for _ in range(contexts)]
        self._held = [0] * contexts
        with torch.inference_mode(False):  # (changed in place later, in whatever mode)
            self.table = torch.full((contexts, self.slots), -1, dtype=torch.int32, device=device)
            self.lengths = torch.zeros(contexts, dtype=torch.int32, device=device)

    @property
    def held(self) -> Tuple[int, ...]:
        """Tokens of each context (on the host)."""
        return tuple(self._held)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _needed(self, counts: Sequence[int]) -> List[int]:
        if len(counts) != len(self._held) or any(int(c) < 0 for c in counts):
            raise ValueError(f"{len(self._held)} counts of zero or more tokens: got {list(counts)}")
        return [-(-(h + int(c)) // self.page_size) for h, c in zip(self._held, counts)]

    def check(self, counts: Sequence[int]) -> None:
        """Raise unless every context can take that many tokens more."""
        need = self._needed(counts)
        over = [b for b, n in enumerate(need) if n > self.slots]
        if over:
            raise RuntimeError(f"contexts {over} would pass {self.slots} pages of {self.page_size} tokens")
        wanted = sum(n - len(p) for n, p in zip(need, self._pages))
        if wanted > len(self._free):
            raise RuntimeError(f"{wanted} pages wanted, {len(self._free)} of {self.num_pages} free: release a context or make the pool larger")

    def extend(self, counts: Sequence[int]) -> Tuple[torch.Tensor, torch.Tensor]:
        """Pages for ``counts[b]`` tokens more of every context.  -> (offsets [contexts + 1], starts [contexts]) of ``append_context``;
        ``lengths`` counts the new tokens from here on.  Raises, and changes nothing, where the pool or a context's slots do not suffice."""
        self._not_captured()
        self.check(counts)
        device = self.table.device
        held, offsets = [h + int(c) for h, c in zip(self._held, counts)], [0]
        rows, cols, ids, free = [], [], [], len(self._free)
        for b, (need, c) in enumerate(zip(self._needed(counts), counts)):
            for slot in range(len(self._pages[b]), need):
                free -= 1
                rows.append(b), cols.append(slot), ids.append(self._free[free])
            offsets.append(offsets[-1] + int(c))
        # everything that can fail first: an error leaves the bookkeeping as it was
        starts, lengths, ends = (torch.tensor(x, dtype=torch.int32).to(device) for x in (self._held, held, offsets))
        if ids:
            self.table[torch.tensor(rows, device=device), torch.tensor(cols, device=device)] = torch.tensor(ids, dtype=torch.int32, device=device)
        self.lengths.copy_(lengths)
        for b, page in zip(rows, ids):
            self._pages[b].append(page)
        del self._free[free:]
        self._held = held
        return ends, starts

    def _take_back(self, held: Sequence[int]) -> None:
        """Every context holds ``held[b]`` tokens again: undoes an ``extend`` whose tokens could not be stored."""
        self.lengths.copy_(torch.tensor(held, dtype=torch.int32))
        for b in reversed(range(len(held))):  # (the pool's order as it was)
            keep = -(-held[b] // self.page_size)
            self.table[b, keep:].fill_(-1)
            self._free.extend(reversed(self._pages[b][keep:]))
            del self._pages[b][keep:]
        self._held = list(held)

    def release(self, context: int) -> None:
        """Forget a context; its pages go back to the pool."""
        self._not_captured()
        self.table[context].fill_(-1)
        self.lengths[context].zero_()
        self._free.extend(reversed(self._pages[context]))
        self._pages[context] = []
        self._held[context] = 0

    def _not_captured(self) -> None:
        if self.table.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the page table is kept on the host: extend and release outside a captured graph (its replays read the new table)")


class LayerContext:
    """One layer's share of a ``ContextMemory``: what an attention layer takes in place of cached keys and values."""

    def __init__(self, memory: "ContextMemory", pages: ContextPages):
        self.memory, self.pages = memory, pages

    def attend(self, q: torch.Tensor, heads: int, empty: Optional[torch.Tensor] = None) -> torch.Tensor:
        """softmax(q k^T / sqrt(head_dim)) v of rotated queries [contexts, T, heads * head_dim] over the memory (over its
        ``selected_pages`` best pages where that is set); 16-bit pages: q is rounded to their type, the result is of q's.
        ``empty`` [heads * head_dim]: the result for a context that holds nothing (zeros unless given)."""
        m, t = self.memory, self.memory.pages_of
        x = q if q.dtype is self.pages.keys.dtype else q.to(self.pages.keys.dtype)
        chosen = None if m.selected_pages is None else select_pages(x, self.pages, t.table, t.lengths, heads, m.selected_pages)
        out = context_attention(x, self.pages, t.table, t.lengths, heads, pages=chosen).to(q.dtype)
        # (the host knows whether there is such a context now; a graph is replayed when there may be)
        if empty is not None and (0 in t._held or torch.cuda.is_current_stream_capturing()):
            out = torch.where((t.lengths > 0)[:, None, None], out, empty.to(out.dtype))
        return out


class ContextMemory:
    """Growing contexts of the attention layers of a stack: one page table, one set of pages per layer.  ``layers[i]`` is layer i's
    ``LayerContext``."""

    def __init__(self, layers: int, contexts: int, num_pages: int, kv_heads: int, head_dim: int, page_size: int = 64,
                 dtype: torch.dtype = torch.float32, slots: Optional[int] = None, selected_pages: Optional[int] = None, device="cuda"):
        if layers < 1 or (selected_pages is not None and selected_pages < 1):
            raise ValueError("layers and selected_pages have to be positive")
        self.pages_of = PageTable(contexts, num_pages, page_size, slots, device)
        self.selected_pages = selected_pages
        self.layers = [LayerContext(self, allocate_pages(num_pages, kv_heads, head_dim, page_size, dtype, device)) for _ in range(layers)]

    @property
    def contexts(self) -> int:
        return self.pages_of.table.shape[0]

    @property
    def held(self) -> Tuple[int, ...]:
        return self.pages_of.held

    def append(self, counts: Sequence[int], keys_values: Sequence[Tuple[torch.Tensor, torch.Tensor]], positions: Optional[torch.Tensor] = None,
               rotary_dim: Optional[int] = None) -> None:
        """``counts[b]`` tokens more of every context: their (keys, values) of each layer, rows in the contexts' order, and positions.
        A call that is refused changes nothing."""
        if len(keys_values) != len(self.layers):
            raise ValueError(f"{len(self.layers)} layers' keys and values: got {len(keys_values)}")
        n = sum(int(c) for c in counts)
        self.pages_of.check(counts)
        for layer, (k, v) in zip(self.layers, keys_values):  # all of it before the table counts the tokens
            if k.dim() != 2 or k.shape[0] != n or v.shape != k.shape:
                raise ValueError(f"keys and values of {n} tokens: got {tuple(k.shape)}, {tuple(v.shape)}")
            _check_rows(layer.pages, k, v, positions, rotary_dim, 10000.0)
        held = self.held
        offsets, starts = self.pages_of.extend(counts)
        try:
            for layer, (k, v) in zip(self.layers, keys_values):
                append_context(layer.pages, k, v, offsets, starts, self.pages_of.table, positions, rotary_dim)
        except Exception:  # (sizes that the library refuses; what an earlier layer stored lies behind the lengths)
            self.pages_of._take_back(held)
            raise

    def release(self, context: int) -> None:
        self.pages_of.release(context)
