"""A paged K/V cache: appends (``fa_paged_append``) and attention against it (``fa_paged_attn``).

The serving side of the package, next to ``flash_attention_decode`` (one contiguous bf16 cache
per sequence).  Pages of ``page_size`` positions live in a pool (num_pages, H_kv, page_size, D);
a block table (B, columns) says which page holds positions ``[c * page_size, (c + 1) *
page_size)`` of each sequence.  The pool is bf16, or 8-bit (``torch.float8_e4m3fn``) with one
fp32 scale for each page and K/V head: value = code * scale.

A step of a server is two calls::

    q = paged_kv_append(cache, table, kv_lens, k, v, new_lens=new, rotary=spec, q=q)
    o, lse = flash_attention_paged(q, cache, table, kv_lens, causal_mask, q_lens=new)

``kv_lens`` counts each sequence with its new tokens and ``new`` the valid ones among the T rows
of a padded batch (None: all T), so row ``i`` of sequence ``b`` sits at position ``kv_lens[b] -
new[b] + i``.  Both calls read the lengths on the device and never wait for it, so one captured
CUDA graph serves every length up to the table's.  A sequence with ``kv_lens`` 0 is an empty
slot of the batch (without ``new`` too).  Page numbers and lengths out of range are reported by
``check_device_status``: an append writes nothing for them, attention hides such a page and cuts such
a length to what there is.  There is no CPU path.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib as L
from .flash_attn import _DTYPES, has_tangent, on_device, status_ptr
from .mask_mod import MaskMod
from .mask_mod import spec_of as mask_spec_of
from .rotary import RotarySpec
from .score_mod import ScoreMod
from .score_mod import spec_of as score_spec_of

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128, 256)
_CACHE_DTYPES = {torch.bfloat16: L.FA_DTYPE_BF16, torch.float8_e4m3fn: L.FA_DTYPE_E4M3}

Lengths = Union[torch.Tensor, Sequence[int]]


class PagedKVCache:
    """The page pools of keys and values and, for 8-bit pools, their scales.

    ``k`` and ``v`` are (num_pages, H_kv, page_size, D) with a contiguous last dimension (a pool
    stored as (num_pages, page_size, H_kv, D) is passed transposed); ``k_scale`` and ``v_scale``
    are contiguous fp32 (num_pages, H_kv), for ``float8_e4m3fn`` pools only.
    """

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                 v_scale: Optional[torch.Tensor] = None):
        if k.dim() != 4 or v.shape != k.shape:
            raise ValueError(f"k and v must be (num_pages, H_kv, page_size, D), got {tuple(k.shape)} and {tuple(v.shape)}")
        if not k.is_cuda or v.device != k.device:
            raise ValueError("a PagedKVCache lives on one CUDA device (there is no CPU path)")
        if k.dtype not in _CACHE_DTYPES or v.dtype != k.dtype:
            raise ValueError(f"k and v must share dtype bf16 or float8_e4m3fn, got {k.dtype}/{v.dtype}")
        n, hkv, ps, d = k.shape
        if ps not in PAGE_SIZES or d not in HEAD_DIMS:
            raise NotImplementedError(f"page size {ps} and head dim {d}: need one of {PAGE_SIZES} and of {HEAD_DIMS}")
        es = k.element_size()
        for t in (k, v):
            st = t.stride()
            if st[3] != 1 or any((s * es) % 16 for s in st[:3]) or t.data_ptr() % 16:
                raise ValueError("pages need a contiguous last dimension, and 16-byte multiples for base and strides")
            if any(s <= 0 for s, m in zip(st, t.shape) if m > 1):
                raise ValueError("pages must not overlap in memory")
        if k.dtype == torch.float8_e4m3fn:
            for t in (k_scale, v_scale):
                if t is None or t.shape != (n, hkv) or t.dtype != torch.float32 or t.device != k.device or not t.is_contiguous():
                    raise ValueError(f"an 8-bit cache needs contiguous fp32 k_scale and v_scale of shape ({n}, {hkv})")
        elif k_scale is not None or v_scale is not None:
            raise ValueError("scales belong to an 8-bit cache")
        self._k, self._v, self._k_scale, self._v_scale = k, v, k_scale, v_scale
        self._fields = (_CACHE_DTYPES[k.dtype], n, hkv, ps, d, k.data_ptr(), *k.stride()[:3], v.data_ptr(),
                        *v.stride()[:3], *((k_scale.data_ptr(), v_scale.data_ptr()) if k_scale is not None else (0, 0)))
        self._shape, self._device = (n, hkv, ps, d), k.device
        self._plans: dict = {}  # by the shape of a call: see _plan
        status_ptr(k.device.index)  # made here, so that a call's capture finds it

    @classmethod
    def empty(cls, num_pages: int, num_kv_heads: int, page_size: int, head_dim: int,
              dtype: torch.dtype = torch.bfloat16, device="cuda") -> "PagedKVCache":
        """A pool of zeroed pages."""
        shape = (num_pages, num_kv_heads, page_size, head_dim)
        pools = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(2)]
        if dtype == torch.float8_e4m3fn:
            pools += [torch.ones(shape[:2], dtype=torch.float32, device=device) for _ in range(2)]
        return cls(*pools)

    k = property(lambda self: self._k)
    v = property(lambda self: self._v)
    k_scale = property(lambda self: self._k_scale)
    v_scale = property(lambda self: self._v_scale)
    page_size = property(lambda self: self._shape[2])

    def gather(self, pages: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """Keys and values of a row of a block table as fp32 (H_kv, positions, D): for looking at a
        cache, not for speed."""
        out = []
        for pool, scale in ((self.k, self.k_scale), (self.v, self.v_scale)):
            x = pool[pages.long()].float()
            if scale is not None:
                x = x * scale[pages.long()][:, :, None, None]
            out.append(x.transpose(0, 1).flatten(1, 2))
        return tuple(out)

    def _packed(self, table: torch.Tensor) -> tuple:
        """The fields of an FaPagedCache."""
        return (*self._fields, table.data_ptr(), table.shape[1], table.stride(0))


_PACK_APPEND, _PACK_ATTN = L.packer(L.FaPagedAppendParams), L.packer(L.FaPagedAttnParams)
_NONE = (0, 0, 0, 0)
_NO_MASK_TABLES = (0,) * 13  # doc_q .. bit_cols of an FaMaskSpec


def _fields(t: torch.Tensor) -> tuple:
    """The fields of an FaTensor."""
    st = t.stride()
    return t.data_ptr(), st[0], st[1], st[2]


def _out_like(t: torch.Tensor) -> torch.Tensor:
    """A dense tensor like `t` with a contiguous last dimension."""
    o = torch.empty_like(t)
    return o if o.stride(3) == 1 else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(3) == 1 else t.contiguous()


def _int32(x: torch.Tensor, dev: torch.device) -> torch.Tensor:
    """x as int32 on `dev`; what does not fit becomes the nearest int32, which is out of range as well."""
    if x.element_size() > 4 or x.dtype is torch.uint32:
        x = x.to(torch.int64).clamp(-(1 << 31), (1 << 31) - 1)
    return x.to(device=dev, dtype=torch.int32).contiguous()


def _lengths(name: str, x: Lengths, B: int, dev: torch.device) -> torch.Tensor:
    if not (isinstance(x, torch.Tensor) and x.dtype is torch.int32 and x.device == dev and x.is_contiguous()):
        x = torch.as_tensor(x)
        if x.is_floating_point() or x.dtype == torch.bool:
            raise ValueError(f"{name} must be integers")
        x = _int32(x, dev)
    if x.shape != (B,):
        raise ValueError(f"{name} must have shape ({B},), got {tuple(x.shape)}")
    return x


def _table(t: torch.Tensor, B: int, dev: torch.device) -> torch.Tensor:
    if t.dim() != 2 or t.shape[0] != B or t.shape[1] == 0:
        raise ValueError(f"block_table must be ({B}, columns), got {tuple(t.shape)}")
    if t.dtype is not torch.int32 and (t.is_floating_point() or t.dtype == torch.bool):
        raise ValueError("block_table must be integers")
    if t.dtype is not torch.int32 or t.device != dev or t.stride(1) != 1:
        t = _int32(t, dev)
    return t


def paged_kv_append(cache: PagedKVCache, block_table: torch.Tensor, kv_lens: Lengths, k: torch.Tensor,
                    v: torch.Tensor, *, new_lens: Optional[Lengths] = None, rotary: Optional[RotarySpec] = None,
                    q: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Write the new keys and values ``k``, ``v`` (B, H_kv, T, D; bf16 or fp32) into the pages of ``cache``.

    Token ``i < new_lens[b]`` goes to position ``kv_lens[b] - new_lens[b] + i``.  With ``rotary``
    the keys are rotated by that position on the way, and so is ``q`` (B, H, T, D), which is
    returned as a new tensor (rows of padding tokens 0); without ``rotary`` a given ``q`` comes
    back as a copy.  Returns None without ``q``.

    8-bit caches: a page's scale becomes the larger of what it is (if it holds earlier positions of
    the sequence) and the least power of two that fits the largest new magnitude; when it grows,
    the positions held are requantised.  Values beyond the 8-bit range (infinities) are stored as
    the largest one.  Positions behind the new tokens are left as they were.  Each written page
    must be listed once in the tables of the batch.
    """
    if k.dim() != 4 or v.shape != k.shape:
        raise ValueError(f"k and v must be (B, H_kv, T, D), got {tuple(k.shape)} and {tuple(v.shape)}")
    B, hkv, T, D = k.shape
    if (hkv, D) != cache._shape[1::2]:
        raise ValueError(f"k{tuple(k.shape)} does not fit pages {cache._shape}")
    dev = cache._device
    if k.device != dev or v.device != dev or (q is not None and q.device != dev):
        raise ValueError("k, v, q and the cache must be on one CUDA device")
    dtype = k.dtype
    if dtype not in _DTYPES or v.dtype != dtype or (q is not None and q.dtype != dtype):
        raise ValueError("q, k, v must share dtype bf16 or fp32")
    if q is not None and (q.dim() != 4 or (q.shape[0], q.shape[2], q.shape[3]) != (B, T, D)):
        raise ValueError(f"shape mismatch q{tuple(q.shape)} k{tuple(k.shape)}")
    if rotary is not None and rotary.head_dim != D:
        raise ValueError(f"head dim {D}, but the rotary_spec is for {rotary.head_dim}")
    if (k.requires_grad or v.requires_grad or (q is not None and q.requires_grad)) and torch.is_grad_enabled():
        raise ValueError("paged_kv_append has no gradient: call it under torch.no_grad()")
    if has_tangent(k, v, q):
        raise ValueError("paged_kv_append has no gradient: its inputs cannot carry tangents")
    out, heads, fq, fo = None, 0, _NONE, _NONE
    if q is not None:
        out = _out_like(q)
    if B == 0 or T == 0:
        return out
    if q is not None and q.shape[1]:
        q = _rows(q)
        heads, fq, fo = q.shape[1], _fields(q), _fields(out)
    k, v = _rows(k), _rows(v)
    table, lens = _table(block_table, B, dev), _lengths("kv_lens", kv_lens, B, dev)
    new = None if new_lens is None else _lengths("new_lens", new_lens, B, dev)
    block = _PACK_APPEND.pack(_DTYPES[dtype], B, heads, T, *fq, *_fields(k), *_fields(v), *fo, lens.data_ptr(),
                              0 if new is None else new.data_ptr(),
                              *(rotary.packed(dev) if rotary is not None else (0, 0, 0, 1.0)), *cache._packed(table),
                              status_ptr(dev.index))
    with on_device(dev) as stream:
        L.packed_call("fa_paged_append", block, stream)
    return out


def _plan(cache: PagedKVCache, B: int, H: int, Tq: int, table: torch.Tensor) -> tuple:
    """(workspace bytes, patterns of lse and of the workspace) for calls of this shape, kept with the cache.
    The patterns are one element expanded: torch.empty_like of them costs less than torch.empty."""
    p = L.FaPagedAttnParams()
    p.B, p.H, p.Tq = B, H, Tq
    c = p.cache
    (c.dtype, c.num_pages, c.H_kv, c.page_size, c.D, c.k.ptr, c.k.stride_b, c.k.stride_h, c.k.stride_t, c.v.ptr,
     c.v.stride_b, c.v.stride_h, c.v.stride_t, c.k_scale, c.v_scale, c.block_table, c.table_cols,
     c.table_stride) = cache._packed(table)
    n = C.c_size_t(0)
    with on_device(cache._device):
        L.check(L.lib().fa_paged_attn_workspace_size(C.byref(p), C.byref(n)))
    if len(cache._plans) >= 256:
        cache._plans.clear()
    plan = (n.value, torch.empty(1, dtype=torch.float32, device=cache._device).expand(B, H, Tq),
            torch.empty(1, dtype=torch.uint8, device=cache._device).expand(n.value))
    cache._plans[(B, H, Tq, table.shape[1])] = plan
    return plan


def flash_attention_paged(q: torch.Tensor, cache: PagedKVCache, block_table: torch.Tensor, kv_lens: Lengths,
                          mask_mod: Optional[MaskMod] = None, *, q_lens: Optional[Lengths] = None,
                          score_mod: Optional[ScoreMod] = None,
                          scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention of ``q`` (B, H, Tq, D) bf16 against the cached positions of each sequence.

    Row ``i < q_lens[b]`` sits at position ``kv_lens[b] - q_lens[b] + i`` (``q_lens`` None: all Tq
    rows), so ``causal_mask`` lets each new token see the cache and the new tokens before it.
    ``mask_mod`` may be None (every cached position), ``causal_mask``, ``sliding_window_mask`` or
    their ``and_masks``; ``score_mod`` ALiBi, softcap or both.  Any Tq: one token of a decode step,
    drafted tokens, a chunk of a prompt.  Returns ``(o, lse)``, ``o`` like ``q`` and ``lse``
    (B, H, Tq) fp32 (natural log); padding rows and rows that see no position give ``o = 0`` and
    ``lse = -inf``, whatever the cache holds.  Rows before position 0 (``q_lens`` above ``kv_lens``) see
    what the mask lets them see, nothing under ``causal_mask``.

    Keys are hidden from a row by its mask alone: a NaN or infinity in a cached value that some row
    of the same sequence and K/V head sees reaches only what it would reach by the formula as long
    as no other row of the call masks that position away.
    """
    if q.dim() != 4:
        raise ValueError("q must be (B, H, Tq, D)")
    dev = cache._device
    if q.device != dev:
        raise ValueError("q and the cache must be on one CUDA device")
    if q.dtype != torch.bfloat16:
        raise ValueError(f"q must be bf16, got {q.dtype}")
    B, H, Tq, D = q.shape
    hkv = cache._shape[1]
    if D != cache._shape[3]:
        raise ValueError(f"q{tuple(q.shape)} does not fit pages {cache._shape}")
    if H == 0 or H % hkv:
        raise ValueError(f"H={H} must be a multiple of the K/V heads {hkv}")
    if q.requires_grad and torch.is_grad_enabled():
        raise ValueError("flash_attention_paged has no gradient: call it under torch.no_grad()")
    if has_tangent(q):
        raise ValueError("flash_attention_paged has no gradient: q cannot carry a tangent")
    mspec = mask_spec_of(mask_mod)
    if mspec is None or mspec.flags & ~(L.FA_MASK_CAUSAL | L.FA_MASK_WINDOW):
        raise NotImplementedError("paged attention takes None, causal_mask, sliding_window_mask or their and_masks")
    sspec = score_spec_of(score_mod)
    if sspec is None or sspec.flags & ~(L.FA_SCORE_ALIBI | L.FA_SCORE_SOFTCAP):
        raise NotImplementedError("paged attention takes alibi_score_mod, softcap_score_mod or their composition")
    if B == 0 or Tq == 0:
        return torch.empty_like(q), torch.empty((B, H, Tq), dtype=torch.float32, device=dev)
    q = _rows(q)
    table, lens = _table(block_table, B, dev), _lengths("kv_lens", kv_lens, B, dev)
    qlen = None if q_lens is None else _lengths("q_lens", q_lens, B, dev)
    plan = cache._plans.get((B, H, Tq, table.shape[1]))
    if plan is None:
        plan = _plan(cache, B, H, Tq, table)
    size, lse_like, ws_like = plan
    o, lse, ws = _out_like(q), torch.empty_like(lse_like), torch.empty_like(ws_like)
    slopes = 0
    if sspec.flags & L.FA_SCORE_ALIBI:
        t = sspec.device_tensors(dev)["slopes"]
        if t.numel() != H:
            raise ValueError(f"ALiBi has {t.numel()} slopes for {H} heads")
        slopes = t.data_ptr()
    block = _PACK_ATTN.pack(B, H, Tq, *_fields(q), *_fields(o), lse.data_ptr(), lens.data_ptr(),
                            0 if qlen is None else qlen.data_ptr(), scale if scale is not None else 1.0 / math.sqrt(D),
                            mspec.flags, mspec.window_left, mspec.window_right, *_NO_MASK_TABLES,
                            sspec.flags, sspec.softcap, slopes, 0, 0, 0, *cache._packed(table), status_ptr(dev.index))
    with on_device(dev) as stream:
        L.packed_call("fa_paged_attn", block, ws.data_ptr(), size, stream)
    return o, lse
