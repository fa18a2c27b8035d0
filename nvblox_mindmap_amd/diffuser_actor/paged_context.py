"""Keys and values of growing contexts in pages, and the attention over them (libmmfusion: mmf_paged_append, mmf_paged_attention,
mmf_paged_select; csrc/mmf_kernels_paged.hip).

The policy's cross-attention (mindmap/diffuser_actor/diffusion_head.py) reads one observation's context, projected anew for every
inference and padded to one length per batch.  Here a context grows: its tokens' keys (rotated by their position on the way in) and
values are kept in pages of ``page_size`` tokens, so contexts of unlike length share one pool without padding, what was seen before
is not projected again, and a long context can be attended to through its few relevant pages.

``ContextPages`` names the buffers of one layer, ``append_context`` / ``context_attention`` / ``select_pages`` are the operators over
them (float32, float16, bfloat16; no autograd; nothing synchronises, all lengths are read on the device, so calls can be captured into
a graph and replayed with other lengths)."""
import functools
from typing import NamedTuple, Optional

import torch

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


def _check(cond: bool, what: str) -> None:
    if not cond:
        raise ValueError(what)


def _check_pages(c: ContextPages, summary: bool) -> None:
    k, v = c.keys, c.values
    _check(k.dim() == 4 and v.dim() == 4, "keys [pages, kv_heads, page_size, W] and values [pages, kv_heads, W, page_size]")
    n, h, p, w = k.shape
    _check(k.dtype in _TYPES and v.dtype == k.dtype, f"pages are float32, float16 or bfloat16, all alike: got {k.dtype}, {v.dtype}")
    _check(p in PAGE_SIZES, f"page_size {p}: one of {PAGE_SIZES}")
    _check(w == head_width(c.head_dim), f"head_dim {c.head_dim} has pages of {head_width(c.head_dim)} channels, not {w}")
    _check(v.shape == (n, h, w, p), f"values {tuple(v.shape)} do not go with keys {tuple(k.shape)}")
    _check(n > 0 and h > 0, "no pages")
    _check(k.is_contiguous() and v.is_contiguous() and k.data_ptr() % 16 == 0 and v.data_ptr() % 16 == 0, "pages are contiguous and 16-byte aligned")
    _check(v.device == k.device, "pages on one device")
    if summary:
        for s in (c.key_min, c.key_max):
            _check(s is not None, "pages without key_min / key_max")
            _check(s.shape == (n, h, w) and s.dtype == k.dtype and s.device == k.device and s.is_contiguous() and s.data_ptr() % 16 == 0,
                   "key_min / key_max [pages, kv_heads, W] of the pages' type, contiguous, 16-byte aligned")


def _check_int(t: torch.Tensor, dim: int, device, name: str) -> None:
    _check(t.dtype == torch.int32 and t.dim() == dim and t.device == device and t.is_contiguous(), f"{name}: a contiguous int32 tensor of {dim} dimension(s) on {device}")


def _check_inputs(device, *ts: Optional[torch.Tensor]) -> None:
    if device.type != "cuda":
        raise RuntimeError("paged contexts live on an MI355X (no CPU fallback)")
    for t in ts:
        if t is not None:
            _check(t.device == device, f"all tensors on {device}: got one on {t.device}")
            if t.requires_grad and torch.is_grad_enabled():
                raise RuntimeError("paged contexts have no backward pass: call them under torch.no_grad(), or detach the inputs")


def _on(device):
    """The device current while a call launches (torch's default where it is already)."""
    return torch.cuda.device(device)


@functools.lru_cache(maxsize=512)
def _attention_bytes(B, T, H, G, hd, capacity, selected) -> int:
    return int(_lib.lib().mmf_paged_attention_workspace_bytes(B, T, H, G, hd, capacity, selected))


def _rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def append_context(context: ContextPages, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor, starts: torch.Tensor, table: torch.Tensor,
                   positions: Optional[torch.Tensor] = None, rotary_dim: Optional[int] = None, rotary_base: float = 10000.0) -> None:
    """Rows ``offsets[b] : offsets[b + 1]`` of k and v [n, kv_heads * head_dim] (the pages' type or float32; rows may be strided) become
    tokens ``starts[b]``, ``starts[b] + 1``, ... of context b, in the pages ``table[b]`` [contexts, slots] names; rows behind
    ``offsets[-1]``, and tokens whose table entry is outside [0, num_pages) or behind the table, are not stored.

    With ``positions`` [n, axes] (float32, 1 to 4 axes) the keys are rotated on the way as ``layers.rotary3d`` / ``apply_rotary`` do:
    ``rotary_dim`` channels, each axis a share of them.  rotary_dim = kv_heads * head_dim (the default): one code over the whole row, the
    policy's; rotary_dim <= head_dim: the first channels of every head.  Angles are taken in 64 bits (far positions keep their fraction).

    A page gets tokens of one context in a call (two that append to one page in the same call leave it undefined); pages that are only
    read may be shared."""
    device = context.keys.device
    _check_inputs(device, k, v, positions)
    _check_pages(context, True)
    n_pages, h, p, _ = context.keys.shape
    row = h * context.head_dim
    _check(k.dim() == 2 and k.shape == v.shape and k.shape[1] == row, f"k and v [n, {row}]: got {tuple(k.shape)}, {tuple(v.shape)}")
    _check(k.dtype == v.dtype and k.dtype in (context.keys.dtype, torch.float32), f"k and v are {context.keys.dtype} or float32, both alike: got {k.dtype}, {v.dtype}")
    _check_int(table, 2, device, "table")
    _check_int(starts, 1, device, "starts")
    _check_int(offsets, 1, device, "offsets")
    b, slots = table.shape
    _check(starts.shape[0] == b and offsets.shape[0] == b + 1, f"{b} contexts have {b} starts and {b + 1} offsets")
    axes, rotary = 1, 0
    if positions is not None:
        _check(positions.dim() == 2 and positions.shape[0] == k.shape[0] and 1 <= positions.shape[1] <= 4 and positions.dtype == torch.float32
               and positions.is_contiguous(), f"positions [{k.shape[0]}, axes] float32, contiguous, 1 to 4 axes")
        axes, rotary = positions.shape[1], row if rotary_dim is None else int(rotary_dim)
        _check(rotary > 0 and rotary % (2 * axes) == 0 and (rotary <= context.head_dim or rotary == row),
               f"rotary_dim {rotary}: a multiple of {2 * axes}, at most head_dim {context.head_dim} or the whole row {row}")
        _check(rotary_base > 0, "rotary_base has to be positive")
    else:
        _check(rotary_dim is None, "rotary_dim without positions")
    if k.shape[0] == 0 or b == 0 or slots == 0:
        return
    k, v = _rows(k), _rows(v)
    with _on(device):
        _lib.check(_lib.lib().mmf_paged_append(_lib.dptr(k), k.stride(0), _lib.dptr(v), v.stride(0), _TYPES[k.dtype], k.shape[0], _lib.dptr(positions), axes,
                                               rotary, float(rotary_base), _lib.dptr(offsets), _lib.dptr(starts), _lib.dptr(table), b, slots, p, h,
                                               context.head_dim, n_pages, _TYPES[context.keys.dtype], _lib.dptr(context.keys), _lib.dptr(context.values),
                                               _lib.dptr(context.key_min), _lib.dptr(context.key_max), _lib.stream_ptr(device)), "mmf_paged_append")


def _check_query(q: torch.Tensor, context: ContextPages, table: torch.Tensor, lengths: torch.Tensor, heads: int):
    device = context.keys.device
    h = context.keys.shape[1]
    _check(heads > 0 and heads % h == 0, f"heads {heads}: a multiple of the {h} key-value heads")
    _check(q.dim() == 3 and q.shape[2] == heads * context.head_dim, f"q [contexts, tokens, {heads * context.head_dim}]: got {tuple(q.shape)}")
    _check(q.dtype == context.keys.dtype, f"q is {q.dtype}, the pages are {context.keys.dtype}")
    _check_int(table, 2, device, "table")
    _check_int(lengths, 1, device, "lengths")
    _check(table.shape[0] == q.shape[0] == lengths.shape[0], f"{q.shape[0]} contexts: table {tuple(table.shape)}, lengths {tuple(lengths.shape)}")


def context_attention(q: torch.Tensor, context: ContextPages, table: torch.Tensor, lengths: torch.Tensor, heads: int,
                      scale: Optional[float] = None, pages: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale q k^T) v per head over the first ``lengths[b]`` tokens of context b (scale: 1 / sqrt(head_dim) unless given); q
    [contexts, T, heads * head_dim] of the pages' type, rotated by the caller (``fused_ops.rotary_apply``, ``q_block``); query head i reads
    key-value head i // (heads / kv_heads).  ``pages`` [contexts, T, kv_heads, count] int32 (``select_pages``): over the tokens of these
    table slots only; an entry outside the table holds nothing, none may stand twice.  Zeros where there is no token.  -> [contexts, T, heads * head_dim]."""
    device = context.keys.device
    _check_inputs(device, q, table, lengths)
    _check_pages(context, False)
    _check_query(q, context, table, lengths, heads)
    n_pages, h, p, _ = context.keys.shape
    b, t, _ = q.shape
    slots, count = table.shape[1], 0
    if pages is not None:
        _check_int(pages, 4, device, "pages")
        _check(pages.shape[:3] == (b, t, h), f"pages [{b}, {t}, {h}, count]: got {tuple(pages.shape)}")
        count = pages.shape[3]
    if q.numel() == 0 or slots == 0 or (pages is not None and count == 0):
        return torch.zeros(q.shape, dtype=q.dtype, device=device)
    q = q.contiguous()
    out = torch.empty_like(q)
    need = _attention_bytes(b, t, h, heads // h, context.head_dim, (slots if pages is None else count) * p, int(pages is not None))
    # per call, from torch's caching allocator: safe inside a captured graph (its private pool) and across streams
    work = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    with _on(device):
        _lib.check(_lib.lib().mmf_paged_attention(_lib.dptr(q), _lib.dptr(context.keys), _lib.dptr(context.values), _TYPES[q.dtype], _lib.dptr(table),
                                                  _lib.dptr(lengths), _lib.dptr(pages), count, b, t, h, heads // h, context.head_dim, slots, n_pages, p,
                                                  context.head_dim ** -0.5 if scale is None else float(scale), _lib.dptr(out), _lib.dptr(work), need,
                                                  _lib.stream_ptr(device)), "mmf_paged_attention")
    return out


def select_pages(q: torch.Tensor, context: ContextPages, table: torch.Tensor, lengths: torch.Tensor, heads: int, count: int) -> torch.Tensor:
    """Table slots of the ``count`` pages that can hold the largest products with each query token, for every key-value head:
    [contexts, T, kv_heads, count] int32, ascending, filled up with -1 -- the ``pages`` of ``context_attention``.  A page's score is
    sum_c max(q_c, 0) key_max_c + min(q_c, 0) key_min_c, which no key of the page exceeds, the largest over the query heads that share the
    key-value head; taken in 64 bits, the lower slot first among equals."""
    device = context.keys.device
    _check_inputs(device, q, table, lengths)
    _check_pages(context, True)
    _check_query(q, context, table, lengths, heads)
    _check(count > 0, "count has to be positive")
    n_pages, h, p, _ = context.keys.shape
    b, t, _ = q.shape
    slots = table.shape[1]
    if q.numel() == 0 or slots == 0:
        return torch.full((b, t, h, count), -1, dtype=torch.int32, device=device)
    q = q.contiguous()
    out = torch.empty((b, t, h, count), dtype=torch.int32, device=device)
    need = 8 * b * t * h * slots
    work = torch.empty(need, dtype=torch.uint8, device=device)
    with _on(device):
        _lib.check(_lib.lib().mmf_paged_select(_lib.dptr(q), _lib.dptr(context.key_min), _lib.dptr(context.key_max), _TYPES[q.dtype], _lib.dptr(table),
                                               _lib.dptr(lengths), b, t, h, heads // h, context.head_dim, slots, n_pages, p, count, _lib.dptr(out),
                                               _lib.dptr(work), need, _lib.stream_ptr(device)), "mmf_paged_select")
    return out
