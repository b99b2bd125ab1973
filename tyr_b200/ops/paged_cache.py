"""A paged K/V cache for batches of ragged sequences: new tokens' keys and values written with their norms and rotation on the way (csrc/paged_append.cu), and
attention over the pages (csrc/paged_attention.cu).

Pages ``[pages, kv heads, page, head size]`` hold ``page`` tokens each, in 16 bits or as e4m3 codes in units of a scale for each (page, head).  Sequence ``b`` has
``lengths[b]`` tokens, the new ones among them, at ``table[b, position // page]``; its new tokens are rows ``starts[b] .. starts[b + 1] - 1`` of the operands and its
last positions.  Without ``starts`` every sequence has one row, and none where its length is 0.  Lengths, starts and table live on the device: a step has no shapes
that depend on them and can be replayed from a CUDA graph.  A page that is written belongs to one sequence and stands in its row of the table once; full pages may be shared.

On the GPU, operands that do not go together (a page outside the cache, a length beyond the table or the rotation) are left out and recorded
(:func:`tyr_b200.ops._common.raise_on_device_error`): nothing is written, the rows of a sequence that is left out are zeros, and those that would see a page outside the
cache are NaN.  The CPU path states the same contract in plain PyTorch, refuses them, and is the oracle of the numerics tests."""
from __future__ import annotations

import ctypes
import functools
import math
import struct
from typing import List, Optional, Tuple

import torch

from .._native import register_signatures
from ._common import check, cur_stream, err_word, lib

E4M3 = torch.float8_e4m3fn
LARGEST = 448.0                     # of e4m3
LEAST_EXPONENT = -100               # of a page's scale
HEAD_SIZES = (64, 128, 256)
PAGE_SIZES = (16, 32, 64, 128)
_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
# capacity up to which the keys of a (sequence, head) are not cut into pieces
WHOLE_MAX_KEYS = 256
# runs of 16 keys of the table's capacity for each share of the work, while there are not more shares than the device holds CTAs at once (a sequence shorter than
# its row of the table leaves its shares less)
LEAST_TILES = 8


@register_signatures
def _sigs(lib_):
    P, I = ctypes.c_void_p, ctypes.c_int
    if hasattr(lib_, "tyr_paged_append"):
        lib_.tyr_paged_append.argtypes, lib_.tyr_paged_append.restype = [P, I, P], I
    if hasattr(lib_, "tyr_paged_attention"):
        lib_.tyr_paged_attention.argtypes, lib_.tyr_paged_attention.restype = [P, I, I, P], I
        lib_.tyr_paged_attention_gathered.argtypes, lib_.tyr_paged_attention_gathered.restype = [P, I, ctypes.c_longlong, P], I
        lib_.tyr_paged_attention_resident.argtypes, lib_.tyr_paged_attention_resident.restype = [I] * 5, I


# the kernels' argument blocks, as csrc/paged_append.cu and csrc/paged_attention.cu declare them
_APPEND = struct.Struct("@16Q7q11if0q")
_ATTEND = struct.Struct("@11Q3q10ifi0q")


class PagedStore:
    """The pages of one layer: ``k`` and ``v`` [pages, kv heads, page, head size] in e4m3, bf16 or fp16, and the scales [pages, kv heads] of e4m3 pages:
    powers of two, as :func:`paged_append` writes them (others may be rounded to the queries' type together with their codes)."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "shape", "index")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None):
        shape, dtype, dev = k.shape, k.dtype, k.get_device()
        if len(shape) != 4 or v.shape != shape or v.dtype != dtype or v.get_device() != dev or not (k.is_contiguous() and v.is_contiguous()):
            raise ValueError("paged store: k and v are contiguous [pages, kv heads, page, head size] of one type and device")
        if (dtype == E4M3) != (k_scale is not None) or (k_scale is None) != (v_scale is None):
            raise ValueError("paged store: e4m3 pages need k_scale and v_scale, other pages have none")
        if k_scale is not None:
            for s in (k_scale, v_scale):
                if s.shape != shape[:2] or s.dtype != torch.float32 or not s.is_contiguous() or s.get_device() != dev:
                    raise ValueError("paged store: scales are contiguous fp32 [pages, kv heads] beside the pages")
        elif dev >= 0 and dtype not in _DTYPES or not dtype.is_floating_point:
            raise ValueError(f"paged store: pages in {dtype} are not supported")
        self.k, self.v, self.k_scale, self.v_scale, self.shape, self.index = k, v, k_scale, v_scale, tuple(shape), dev

    @staticmethod
    def allocate(pages: int, kv_heads: int, page: int, head_dim: int, device, dtype: torch.dtype = E4M3) -> "PagedStore":
        if min(pages, kv_heads, page, head_dim) <= 0:
            raise ValueError("paged store: sizes must be positive")
        k, v = (torch.zeros((pages, kv_heads, page, head_dim), dtype=dtype, device=device) for _ in range(2))
        if dtype != E4M3:
            return PagedStore(k, v)
        return PagedStore(k, v, *(torch.full((pages, kv_heads), 2.0 ** LEAST_EXPONENT, dtype=torch.float32, device=device) for _ in range(2)))

    @property
    def page(self) -> int:
        return self.shape[2]

    def values(self, pages: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """What these pages hold, fp32 [len(pages), kv heads, page, head size] of the keys and of the values."""
        k, v = self.k[pages].float(), self.v[pages].float()
        if self.k_scale is None:
            return k, v
        return k * self.k_scale[pages][..., None, None], v * self.v_scale[pages][..., None, None]

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scale, self.v_scale) if t is not None)


def _together(what: str, store: PagedStore, rows: int, table: torch.Tensor, lengths: torch.Tensor, starts: Optional[torch.Tensor]) -> Tuple[int, int, int]:
    """(sequences, pages of a row of the table, elements between its rows)."""
    shape, stride, size = table.shape, table.stride(), lengths.shape
    if len(size) != 1 or size[0] == 0 or lengths.dtype != torch.int32 or not lengths.is_contiguous():
        raise ValueError(f"{what}: lengths are contiguous int32 [sequences]")
    B = size[0]
    if len(shape) != 2 or shape[0] != B or shape[1] == 0 or table.dtype != torch.int32 or (stride[1] != 1 and shape[1] > 1):
        raise ValueError(f"{what}: the table is int32 [sequences, pages] with contiguous rows")
    if starts is None:
        if rows != B:
            raise ValueError(f"{what}: {rows} rows for {B} sequences need starts")
    elif starts.shape != (B + 1,) or starts.dtype != torch.int32 or not starts.is_contiguous():
        raise ValueError(f"{what}: starts are contiguous int32 [sequences + 1]")
    dev = store.index
    if table.get_device() != dev or lengths.get_device() != dev or (starts is not None and starts.get_device() != dev):
        raise ValueError(f"{what}: store, table, lengths and starts lie on different devices")
    return B, shape[1], stride[0]


def _on_gpu(what: str, store: PagedStore, dtype: torch.dtype) -> int:
    """The kernels' number of the operands' type; refuses what they do not serve."""
    _, _, P, D = store.shape
    number = _DTYPES.get(dtype)
    if number is None or (store.k_scale is None and store.k.dtype != dtype):
        raise ValueError(f"{what}: operands in {dtype} over pages in {store.k.dtype} are not supported")
    if D not in HEAD_SIZES or P not in PAGE_SIZES:
        raise ValueError(f"{what}: heads of {D} in pages of {P} are not supported (heads of {HEAD_SIZES}, pages of {PAGE_SIZES})")
    if (store.k.data_ptr() | store.v.data_ptr()) & 15:
        raise ValueError(f"{what}: pages must lie at multiples of 16 bytes")
    return number


def _rows_of(t: torch.Tensor) -> torch.Tensor:
    """``t`` [rows, heads, D] as the kernels read it: whole heads, 16-byte aligned."""
    row, head, one = t.stride()
    return t if one == 1 and (row | head) & 7 == 0 and t.data_ptr() & 15 == 0 else t.clone(memory_format=torch.contiguous_format)


def _aligned(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    if t.dtype != dtype:
        t = t.to(dtype)
    return t if t.is_contiguous() and t.data_ptr() & 15 == 0 else t.clone(memory_format=torch.contiguous_format)


def _spans(what: str, store: PagedStore, rows: int, table, lengths, starts) -> List[Tuple[int, int, int, List[int]]]:
    """CPU: (first row, rows, length, pages) of every sequence, refusing what does not go together."""
    lens = lengths.tolist()
    at = list(range(rows + 1)) if starts is None else starts.tolist()
    out, P = [], store.page
    for b, n in enumerate(lens):
        new = at[b + 1] - at[b] if starts is not None else int(n > 0)
        if new < 0 or at[b] < 0 or at[b] + new > rows or n < new:
            raise ValueError(f"{what}: sequence {b} has rows {at[b]} to {at[b + 1]} of {rows} and {n} tokens")
        need = -(-n // P) if new else 0
        if need > table.shape[1]:
            raise ValueError(f"{what}: sequence {b} has {n} tokens and {table.shape[1]} pages of {P}")
        pages = table[b, :need].tolist()
        if any(not 0 <= p < store.k.shape[0] for p in pages):
            raise ValueError(f"{what}: sequence {b} names a page outside the {store.k.shape[0]} of the cache")
        out.append((at[b], new, n, pages))
    return out


def _turned(x: torch.Tensor, weight, cos, sin, eps: float, one_plus_w: bool) -> torch.Tensor:
    """Norm, then rotation of channels (i, i + half), rounded nowhere; x: [rows, heads, D], cos / sin: [rows, half]."""
    x = x if x.dtype == torch.float64 else x.float()
    if weight is not None:
        w = weight.to(x.dtype) + (1.0 if one_plus_w else 0.0)
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w
    if cos is None:
        return x
    half, c, s = cos.shape[-1], cos.to(x.dtype)[:, None], sin.to(x.dtype)[:, None]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * c - b * s, a * s + b * c, x[..., 2 * half:]], -1)


def page_scale(amax: torch.Tensor) -> torch.Tensor:
    """2^e with the smallest e >= LEAST_EXPONENT that keeps magnitudes up to ``amax`` within e4m3; NaN where one is not finite."""
    m, x = torch.frexp(amax.float())
    e = torch.where(amax > 0, x - 9 + (m > 0.875).int(), LEAST_EXPONENT).clamp_min(LEAST_EXPONENT)
    return torch.where(torch.isfinite(amax), torch.ldexp(torch.ones_like(m), e), math.nan)


def _append_ref(store, k, v, table, lengths, starts, q, cos, sin, q_weight, k_weight, eps, one_plus_w):
    rows, P = k.shape[0], store.page
    spans = _spans("paged_append", store, rows, table, lengths, starts)
    if cos is not None and any(new and n > cos.shape[0] for _, new, n, _ in spans):
        raise ValueError(f"paged_append: a position lies outside the {cos.shape[0]} of the rotation")
    out = None if q is None else torch.zeros_like(q, memory_format=torch.contiguous_format)
    for row, new, n, pages in spans:
        c, s = (None, None) if cos is None else (cos[n - new:n], sin[n - new:n])
        if q is not None:
            out[row:row + new] = _turned(q[row:row + new], q_weight, c, s, eps, one_plus_w).to(q.dtype)
        fresh = (_turned(k[row:row + new], k_weight, c, s, eps, one_plus_w), v[row:row + new])
        for j in range((n - new) // P, -(-n // P) if new else 0):
            lo, hi, page = max(n - new, j * P), min(n, (j + 1) * P), pages[j]
            for x, kept, scales in zip(fresh, (store.k, store.v), (store.k_scale, store.v_scale)):
                x, held = x[lo - n + new:hi - n + new].transpose(0, 1), lo - j * P
                if scales is not None:
                    x = x.float()
                    scale = page_scale(x.abs().amax((1, 2)))
                    if held:
                        scale = torch.maximum(scale, scales[page])              # NaN where either is
                        grown = (scale > scales[page])[:, None, None]
                        old = kept[page, :, :held]
                        moved = (old.float() * (scales[page] / scale)[:, None, None]).to(kept.dtype)
                        kept[page, :, :held] = torch.where(grown, moved.float(), old.float()).to(kept.dtype)
                    scales[page] = scale
                    x = torch.where(torch.isnan(scale)[:, None, None], 0.0, x / scale[:, None, None])
                kept[page, :, held:hi - j * P] = x.to(kept.dtype)
    return out


def paged_append(store: PagedStore, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, starts: Optional[torch.Tensor] = None, *,
                 q: Optional[torch.Tensor] = None, cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, one_plus_w: bool = False) -> Optional[torch.Tensor]:
    """Writes the new tokens' keys and values ``[rows, kv heads, D]`` into their pages and returns the queries ``[rows, heads, D]`` (when given) as attention takes
    them; rows of no sequence come back as zeros.

    Keys and queries get their RMS norm over the head (with ``k_weight`` / ``q_weight`` [D] of their type, ``1 + weight`` with ``one_plus_w``), then channels ``i`` and ``i + half``
    are turned by the row's position (``cos``, ``sin`` fp32 [positions, half]), in 32 bits with one rounding at the end.  Operands may be strided views.

    e4m3 pages: the scale of a (page, head) is the smallest power of two, 2^-100 at least, that keeps its largest magnitude within 448.  It grows with later tokens of
    the page, whose older codes are rescaled (exactly, unless they leave e4m3's normal range); the first slot of a page starts it anew.  A value that is not finite
    makes it NaN until then, and so the attention of all that sees the page."""
    pages, G, P, D = store.shape
    shape, dtype, dev = k.shape, k.dtype, store.index
    if len(shape) != 3 or v.shape != shape or v.dtype != dtype or shape[1] != G or shape[2] != D or shape[0] == 0:
        raise ValueError(f"paged_append: k {tuple(k.shape)} and v {tuple(v.shape)} do not fit pages {store.shape}")
    rows = shape[0]
    if k.get_device() != dev or v.get_device() != dev:
        raise ValueError("paged_append: k, v and the store lie on different devices")
    B, width, table_row = _together("paged_append", store, rows, table, lengths, starts)
    H = 0
    if q is not None:
        size = q.shape
        if len(size) != 3 or size[0] != rows or size[2] != D or size[1] == 0 or q.dtype != dtype or q.get_device() != dev:
            raise ValueError(f"paged_append: queries {tuple(size)} do not fit keys {tuple(shape)}")
        H = size[1]
    if (cos is None) != (sin is None):
        raise ValueError("paged_append: cos and sin go together")
    half = positions = 0
    if cos is not None:
        size = cos.shape
        if len(size) != 2 or sin.shape != size or size[0] == 0 or size[1] == 0 or 2 * size[1] > D or cos.get_device() != dev or sin.get_device() != dev:
            raise ValueError(f"paged_append: cos {tuple(size)} and sin {tuple(sin.shape)} do not fit heads of {D}")
        positions, half = size
    for w in (q_weight, k_weight):
        if w is not None and (w.shape != (D,) or w.dtype != dtype or w.get_device() != dev):
            raise ValueError(f"paged_append: norm weights are {dtype} [{D}] beside the pages")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, cos, sin, q_weight, k_weight)):
        raise ValueError("paged_append: serves inference and has no gradient")
    if dev < 0:
        return _append_ref(store, k, v, table, lengths, starts, q, cos, sin, q_weight, k_weight, eps, one_plus_w)
    number = _on_gpu("paged_append", store, dtype)
    if half % 4:
        raise ValueError(f"paged_append: the rotation turns a multiple of 8 channels, got {2 * half}")
    k, v = _rows_of(k), _rows_of(v)
    (k_row, k_head, _), (v_row, v_head, _) = k.stride(), v.stride()
    cos_at = sin_at = q_weight_at = k_weight_at = q_at = out_at = q_row = q_head = 0
    if half:
        cos, sin = _aligned(cos, torch.float32), _aligned(sin, torch.float32)
        cos_at, sin_at = cos.data_ptr(), sin.data_ptr()
    if k_weight is not None:
        k_weight = _aligned(k_weight, dtype)
        k_weight_at = k_weight.data_ptr()
    out = None
    if q is not None:
        if q_weight is not None:
            q_weight = _aligned(q_weight, dtype)
            q_weight_at = q_weight.data_ptr()
        q = _rows_of(q)
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        q_at, out_at, (q_row, q_head, _) = q.data_ptr(), out.data_ptr(), q.stride()
    k_scale_at = v_scale_at = 0
    if store.k_scale is not None:
        k_scale_at, v_scale_at = store.k_scale.data_ptr(), store.v_scale.data_ptr()
    device = k.device
    packed = _APPEND.pack(q_at, k.data_ptr(), v.data_ptr(), out_at, store.k.data_ptr(), store.v.data_ptr(), k_scale_at, v_scale_at, table.data_ptr(), lengths.data_ptr(),
                          0 if starts is None else starts.data_ptr(), cos_at, sin_at, q_weight_at, k_weight_at, err_word(device).data_ptr(), q_row, q_head, k_row, k_head,
                          v_row, v_head, table_row, rows, B, H, G, D, P, pages, width, positions, half, one_plus_w, eps)
    check(lib().tyr_paged_append(packed, number, cur_stream(device)), "paged_append")
    return out


# the most that keys and values laid out for the kernel on tcgen05 may take
GATHER_MAX_BYTES = 2 ** 30


def gathers(dtype: torch.dtype, f8: bool, rows: int, sequences: int, heads: int, kv_heads: int, D: int, capacity: int, scale: float) -> bool:
    """Whether the pages are laid out for the tensor core's kernel first.  It serves heads of 64 and 128 and numbers of the queries' type (a code times its page's scale
    may leave fp16's range), and takes 128 or 256 rows of one head against 128 keys in 2.5 us an SM, however few rows there are; the other kernel multiplies at 140
    TFLOP/s.  In us a key of context, with the pages' way at 5 TB/s; measured, other / this, 3000 tokens of context: 6 sequences, 20 heads of 128, 32 / 64 / 256
    new tokens each 72 / 64, 98 / 65, 273 / 77; 16, 48 heads 264 / 357, 418 / 364, 1476 / 428; 2, 10 heads 38 / 59, 40 / 60, 67 / 68."""
    if D > 128 or not scale > 0 or (f8 and dtype == torch.float16) or sequences > 65535 or 4 * sequences * kv_heads * (capacity + 127) * D > GATHER_MAX_BYTES:
        return False
    blocks = sequences * -(-rows // (256 * sequences)) * heads
    return max(1.0, blocks / 148) * 2.5 / 128 + sequences * kv_heads * D * (6 if f8 else 8) / 5e6 < rows * heads * D * 4 / 1.4e8


@functools.lru_cache(maxsize=256)
def _resident(index: int, number: int, f8: bool, D: int, tile: int, few: bool) -> int:
    """CTAs of a form of the kernel that device ``index`` holds at once: the shares that a call's work is cut into."""
    cur_stream(torch.device("cuda", index))
    n = lib().tyr_paged_attention_resident(number, f8, D, tile, few)
    if n <= 0:
        raise RuntimeError(f"tyr_b200 native call paged_attention_resident failed with code {n}")
    return n


def _attend_ref(q, store, table, lengths, starts, window, scale):
    rows, H, D = q.shape
    G, wide = store.k.shape[1], torch.float64 if q.dtype == torch.float64 else torch.float32
    out = torch.zeros((rows, H, D), dtype=q.dtype, device=q.device)
    for row, new, n, pages in _spans("paged_attention", store, rows, table, lengths, starts):
        if not new:
            continue
        k, v = (t.to(wide).transpose(0, 1).reshape(G, -1, D)[:, :n] for t in store.values(torch.tensor(pages)))
        s = torch.einsum("ngrd,gld->grnl", q[row:row + new].to(wide).reshape(new, G, H // G, D), k) * scale
        if store.v_scale is not None:                    # a page whose values hold no numbers shows at the keys that are seen, as in the kernel
            s, v = s.masked_fill(torch.isnan(v[..., 0])[:, None, None], math.nan), torch.nan_to_num(v, nan=0.0)
        ago = torch.arange(n - new, n)[:, None] - torch.arange(n)
        unseen = (ago < 0) | (ago >= (window or n))
        s = s.masked_fill(unseen, -math.inf)
        odd = ~torch.isfinite(v)
        o = torch.einsum("grnl,gld->ngrd", s.softmax(-1), v.masked_fill(odd, 0.0))
        for g, key in odd.any(-1).nonzero().tolist():      # values that are not finite show at the rows that see them, and at no others
            o[~unseen[:, key], g] += torch.where(odd[g, key], v[g, key], 0.0)
        out[row:row + new] = o.reshape(new, H, D).to(q.dtype)
    return out


def paged_attention(q: torch.Tensor, store: PagedStore, table: torch.Tensor, lengths: torch.Tensor, starts: Optional[torch.Tensor] = None, *,
                    window: Optional[int] = None, scale: Optional[float] = None) -> torch.Tensor:
    """Attention of the new tokens' queries ``[rows, heads, D]`` over their sequences' pages, which hold the new tokens already -> ``[rows, heads, D]``; rows of no
    sequence, and of one that is left out, come back as zeros.  Scores and sums are held in 32 bits, a probability is rounded once: to the pages' 16-bit type, to f16 beside
    e4m3, or to the queries' type where many new tokens take the kernel on tcgen05 (:func:`gathers`).  Values that are not finite show in their channel at the rows that see
    them.  A token sees the positions up to its own, the last ``window`` of them when given; query heads share K/V heads in groups."""
    pages, G, P, D = store.shape
    shape = q.shape
    if len(shape) != 3 or shape[0] == 0 or shape[2] != D or shape[1] == 0 or shape[1] % G or q.get_device() != store.index:
        raise ValueError(f"paged_attention: queries {tuple(shape)} on {q.device} do not fit pages {store.shape} on {store.k.device}")
    rows, H, _ = shape
    if q.requires_grad and torch.is_grad_enabled():
        raise ValueError("paged_attention: serves inference and has no gradient")
    if window is not None and window <= 0:
        raise ValueError(f"paged_attention: the window must be positive, got {window}")
    B, width, table_row = _together("paged_attention", store, rows, table, lengths, starts)
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    if store.index < 0:
        return _attend_ref(q, store, table, lengths, starts, window, scale)
    dtype, device = q.dtype, q.device
    number = _on_gpu("paged_attention", store, dtype)
    q, f8 = _rows_of(q), store.k_scale is not None
    stride, R = q.stride(), H // G
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if starts is not None and gathers(dtype, f8, rows, B, H, G, D, width * P, scale):
        capacity = -(-width * P // 128) * 128
        numbers = B * G * capacity * D                # keys, values, room for values that are not finite, and a byte for 256 of them
        work = torch.empty(3 * numbers + numbers // 512, dtype=dtype, device=device)
        packed = _ATTEND.pack(q.data_ptr(), out.data_ptr(), store.k.data_ptr(), store.v.data_ptr(), store.k_scale.data_ptr() if f8 else 0, store.v_scale.data_ptr() if f8 else 0,
                              table.data_ptr(), lengths.data_ptr(), starts.data_ptr(), work.data_ptr(), err_word(device).data_ptr(), stride[0], stride[1], table_row, rows, B, H, G,
                              D, P, pages, width, min(window or 0, 2 ** 30), 0, scale, 0)
        check(lib().tyr_paged_attention_gathered(packed, number, capacity, cur_stream(device)), "paged_attention")
        return out
    tile = (64 if D == 256 else 128) if starts is not None and rows * R > 16 * B else 16
    whole = width * P <= WHOLE_MAX_KEYS
    work = None
    if not whole:
        row_tiles = rows * R // tile + B if starts is not None else B * -(-R // tile)
        ctas = min(-(-row_tiles * G * -(-width * P // 16) // LEAST_TILES), _resident(store.index, number, f8, D, tile, starts is None and R <= 8))
        work = torch.empty(ctas * (8 + 2 * tile * (4 + D)), dtype=torch.float32, device=device)
    packed = _ATTEND.pack(q.data_ptr(), out.data_ptr(), store.k.data_ptr(), store.v.data_ptr(), store.k_scale.data_ptr() if f8 else 0, store.v_scale.data_ptr() if f8 else 0,
                          table.data_ptr(), lengths.data_ptr(), 0 if starts is None else starts.data_ptr(), 0 if whole else work.data_ptr(), err_word(device).data_ptr(),
                          stride[0], stride[1], table_row, rows, B, H, G, D, P, pages, width, min(window or 0, 2 ** 30), whole, scale, 0 if whole else ctas)
    check(lib().tyr_paged_attention(packed, number, tile, cur_stream(device)), "paged_attention")
    return out
