"""Keys and values held in 8 bits.

A token's key (or value) of one kv head is held as e4m3 codes times a power of two ``2^e`` of its own, the smallest with
which the row's largest magnitude stays within 448: ``e = ceil(log2(max |x| / 448))``, at least -126; the scale byte is
``e + 127``.  e4m3 rounds relative to a number's own size (half a step is 2^-4 of it; magnitudes below 2^-6 of a code's unit
are held to 2^-10 of the unit), so a power of two loses nothing against a finer scale, and scaling and its undoing are exact
(in bfloat16: from 2^-126 on, and below 2^128, which a row's largest numbers may be rounded to from 248 * 2^120 on).  A row
that holds something that is no finite number is held as NaN throughout.

The codes of sixteen keys lie together in pieces of 64 elements (a last piece of 32 where 64 does not divide the head), each
piece in the order in which the lanes of a matrix instruction take it (:func:`places`): every load of the attention kernel
is one contiguous piece of memory whatever the page size.
"""
from __future__ import annotations

import dataclasses

import torch

KV_DTYPES = ("float8_e4m3",)  # what a cache of keys and values may be held in beside the run dtype
HEAD_DIMS = (32, 64, 96, 128, 256)
MOST_GROUPED = 32  # query heads that may share a kv head
NAN_CODE = 0x7F


def check_kv_dtype(kv_dtype) -> None:
    if kv_dtype is not None and kv_dtype not in KV_DTYPES:
        raise ValueError(f"a cache of keys and values is held in the run dtype (None) or in {', '.join(KV_DTYPES)}, "
                         f"not in {kv_dtype!r}")


def check_page_size(page_size: int) -> None:
    if page_size < 16 or page_size % 16:
        raise ValueError(f"a cache in 8 bits takes pages of a multiple of 16 tokens, not {page_size}")


def check_sizes(num_heads: int, num_kv_heads: int, head_dim: int, page_size: int) -> None:
    """Raises ``ValueError`` for heads or pages that a cache in 8 bits does not take."""
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"a cache in 8 bits takes heads of {', '.join(map(str, HEAD_DIMS))} elements, not {head_dim}")
    check_page_size(page_size)
    if num_kv_heads < 1 or num_heads % num_kv_heads or num_heads // num_kv_heads > MOST_GROUPED:
        raise ValueError(f"a cache in 8 bits takes up to {MOST_GROUPED} query heads on each kv head, not {num_heads} on "
                         f"{num_kv_heads}")


@dataclasses.dataclass(frozen=True)
class QuantizedPages:
    """``codes``: uint8 ``[pages, kv_heads, 2, page_size, head_dim]`` (the last two in :func:`places`' order, sixteen keys
    after sixteen), ``scales``: uint8 ``[pages, kv_heads, 2, page_size]``; index 0 holds keys, 1 values.  ``shape`` is that of
    pages in the run dtype, ``[pages, 2, kv_heads, page_size, head_dim]``."""

    codes: torch.Tensor
    scales: torch.Tensor

    def __post_init__(self):
        c, s = self.codes, self.scales
        if c.dtype != torch.uint8 or s.dtype != torch.uint8 or c.dim() != 5 or c.shape[2] != 2 or s.shape != c.shape[:-1]:
            raise ValueError("pages in 8 bits are uint8 codes [pages, kv_heads, 2, page_size, head_dim] and uint8 scales "
                             f"[pages, kv_heads, 2, page_size], not {c.dtype} {tuple(c.shape)} and {s.dtype} {tuple(s.shape)}")
        if c.device != s.device or not c.is_contiguous() or not s.is_contiguous():
            raise ValueError("the codes and scales of pages in 8 bits are contiguous and on one device")
        p, hk, two, ps, dh = c.shape
        object.__setattr__(self, "shape", torch.Size((p, two, hk, ps, dh)))
        object.__setattr__(self, "device", c.device)

    @classmethod
    def empty(cls, num_pages: int, kv_heads: int, page_size: int, head_dim: int, device, poison: bool = False):
        """Pages of zeros, or (``poison``) of what reads as NaN."""
        check_sizes(kv_heads, kv_heads, head_dim, page_size)
        fill = NAN_CODE if poison else 0  # (as a scale byte: 1)
        new = lambda *shape: torch.full((num_pages, kv_heads, 2, page_size, *shape), fill, dtype=torch.uint8, device=device)
        return cls(new(head_dim), new())

    def poison_(self, pages: torch.Tensor) -> None:
        """What the given pages hold reads as NaN from now on."""
        for t in (self.codes, self.scales):
            t.index_fill_(0, pages, NAN_CODE)


def bytes_per_row(head_dim: int) -> int:
    """A key's (or value's) codes and scale byte."""
    return head_dim + 1


# ------------------------------------------------------------------------------------------------ the plain statement
def places(head_dim: int, device=None):
    """Where element ``d`` of key ``j`` of sixteen lies among their ``16 * head_dim`` codes, ``[16, head_dim]``: keys, values."""
    j = torch.arange(16, device=device)[:, None]
    d = torch.arange(head_dim, device=device)[None, :]
    u = torch.where(head_dim - (d & ~63) >= 64, 16, 8)  # codes that a lane takes
    e, start = d & 63, (d & ~63) * 16
    return start + e // u * 16 * u + j * u + e % u, start + (j >> 2) * 16 * u + (d & 15) * u + (e >> 4) * 4 + (j & 3)


def quantize_rows(x: torch.Tensor):
    """Rows ``[..., head_dim]`` as codes (uint8, element by element) and scale bytes ``[...]``."""
    x = x.float()
    top = x.abs().amax(-1)
    finite = torch.isfinite(x).all(-1)
    m, e = torch.frexp(torch.where(finite, top, torch.zeros_like(top)))  # top = m 2^e, 448 = 0.875 * 2^9
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(min=-126)
    e = torch.where((top > 0) & finite, e, torch.where(finite, -126, 0)).to(torch.int32)
    codes = torch.ldexp(x, -e.unsqueeze(-1)).to(torch.float8_e4m3fn).view(torch.uint8)
    return torch.where(finite.unsqueeze(-1), codes, NAN_CODE).to(torch.uint8), (e + 127).to(torch.uint8)


def store_rows(kv: QuantizedPages, k: torch.Tensor, v: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """Keys and values ``[n, kv_heads, head_dim]`` into their places; a slot that is none is left out."""
    p, _, hk, ps, dh = kv.shape
    slot = slot_mapping.long()
    there = (slot >= 0) & (slot < p * ps)
    slot = slot[there]
    flat = kv.codes.view(p, hk, 2, ps * dh)
    head = torch.arange(hk, device=slot.device)
    for which, x in ((0, k[there]), (1, v[there])):
        codes, byte = quantize_rows(x)
        kv.scales[slot // ps, :, which, slot % ps] = byte
        at = places(dh, slot.device)[which][slot % 16] + ((slot % ps) // 16 * 16 * dh)[:, None]
        flat[(slot // ps)[:, None, None], head[None, :, None], which, at[:, None, :]] = codes


def read_rows(kv: QuantizedPages, page_ids: torch.Tensor):
    """Keys and values of the given pages in float32, ``[n, kv_heads, page_size, head_dim]`` each; a page id that is none
    gives NaN."""
    p, _, hk, ps, dh = kv.shape
    ids = page_ids.long()
    there = (ids >= 0) & (ids < p)
    ids = torch.where(there, ids, 0)
    n = ids.numel()
    codes = kv.codes[ids].view(torch.float8_e4m3fn).float().view(n, hk, 2, ps // 16, 16 * dh)
    scale = torch.ldexp(torch.ones((), device=codes.device), kv.scales[ids].int() - 127).unsqueeze(-1)
    out = []
    for which, at in enumerate(places(dh, codes.device)):
        x = codes[:, :, which][..., at].reshape(n, hk, ps, dh) * scale[:, :, which]
        out.append(torch.where(there.view(n, 1, 1, 1), x, float("nan")))
    return out


def read_pages(kv: QuantizedPages, page_ids: torch.Tensor, dtype=torch.bfloat16) -> torch.Tensor:
    """The given pages in the run dtype's layout: ``[n, 2, kv_heads, page_size, head_dim]`` in memory, a page's values with
    its tokens side by side."""
    k, v = read_rows(kv, page_ids)
    return torch.stack([k, v.transpose(-1, -2).reshape(v.shape)], dim=1).to(dtype)
