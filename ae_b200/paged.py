"""Paged key/value cache of the verify step: append with rotary positions, tree attention.

The MoE layer is one half of a decoder layer; this module is what the other half needs next to
its projections (``specmoe/models/mixtral.py:118-224`` with the pools of
``specmoe/backend/memory.py`` and the backends of ``specmoe/layers/attention_backend/``):

* :func:`kv_append`: norm of each head (optional), rotary positions, and the write of keys and
  values into cache pages, in one launch;
* :func:`paged_attention`: attention of the new tokens over the cached keys, causal or under a
  draft tree's mask, for one new token, a draft tree or a prefill chunk;
* :func:`kv4_read`: rows of a 4-bit cache as 16-bit values.

A cache is two tensors (keys, values) of the same shape and strides,
``[num_pages, kv_heads, page_size, head_dim]`` in the storage dtype, or
``[num_pages, kv_heads, page_size, kv4_row_bytes(head_dim)]`` uint8 for a 4-bit cache
(:func:`new_cache`).  The first three dimensions may have any strides of whole 16 bytes: a
token-major pool ``[num_pages, page_size, kv_heads, head_dim]`` is passed as its
``transpose(1, 2)``.  A token's slot is ``page * page_size + place in the page``.

Everything is for inference (no gradients) and runs on the current stream of the tensors' device.
"""
from __future__ import annotations

import ctypes
import math
from typing import List, Optional, Sequence, Tuple

import torch

from . import _native, ops
from .ops import _STORAGE, _stream_ptr

HEAD_DIMS = (64, 128, 256)


def kv4_row_bytes(head_dim: int) -> int:
    """Bytes of one head's row in a 4-bit cache: codes, then a (scale, zero) pair for each 32
    dims, padded to 16 bytes."""
    if head_dim not in HEAD_DIMS:
        raise NotImplementedError(f"head_dim {head_dim} (supported: {HEAD_DIMS})")
    return -(-(head_dim // 2 + head_dim // 8) // 16) * 16


def new_cache(num_pages: int, kv_heads: int, page_size: int, head_dim: int, dtype: torch.dtype, device,
              bits: int = 16) -> Tuple[torch.Tensor, torch.Tensor]:
    """Zeroed key and value arrays of one layer (``bits`` 16 or 4)."""
    if bits == 16:
        ops.storage_code(dtype)
        if head_dim not in HEAD_DIMS:
            raise NotImplementedError(f"head_dim {head_dim} (supported: {HEAD_DIMS})")
        shape, kind = (num_pages, kv_heads, page_size, head_dim), dtype
    elif bits == 4:
        shape, kind = (num_pages, kv_heads, page_size, kv4_row_bytes(head_dim)), torch.uint8
    else:
        raise NotImplementedError(f"cache of {bits} bits (supported: 16, 4)")
    return torch.zeros(shape, dtype=kind, device=device), torch.zeros(shape, dtype=kind, device=device)


def rope_inv_freq(rot: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                  trained: int = 8192, beta_fast: float = 32.0, beta_slow: float = 1.0,
                  low_freq_factor: float = 1.0, high_freq_factor: float = 4.0,
                  device=None) -> Tuple[torch.Tensor, float]:
    """(``inv_freq`` float64 [rot / 2], ``rope_scale``) for :func:`kv_append`.

    f_i = base^(-2 i / rot), then, for contexts ``factor`` times the ``trained`` length:

    * ``"linear"``: f_i / factor;
    * ``"ntk"``: base * factor^(rot / (rot - 2)) in the place of base;
    * ``"yarn"``: f_i where a pair turns more than ``beta_fast`` times within the trained length,
      f_i / factor below ``beta_slow`` turns, a linear ramp over i between; cos and sin are
      multiplied by 0.1 ln(factor) + 1;
    * ``"llama3"``: f_i above ``high_freq_factor`` turns, f_i / factor below ``low_freq_factor``, a
      ramp linear in the turns between.
    """
    if rot < 0 or rot % 16:
        raise ValueError(f"rot must be a multiple of 16, got {rot}")
    if scaling is not None and factor <= 0:
        raise ValueError("factor must be positive")
    i = torch.arange(rot // 2, dtype=torch.float64)
    if scaling == "ntk" and rot > 2:
        base = base * factor ** (rot / (rot - 2))
    f = torch.pow(torch.tensor(float(base), dtype=torch.float64), -2.0 * i / max(rot, 1))
    scale = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        def index_of(turns):  # the pair that turns so often within the trained length
            return rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(index_of(beta_fast)), 0), min(math.ceil(index_of(beta_slow)), rot - 1)
        stretch = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        f = f * (1 - stretch) + f / factor * stretch
        scale = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    elif scaling == "llama3":
        turns = trained * f / (2 * math.pi)
        keep = ((turns - low_freq_factor) / (high_freq_factor - low_freq_factor)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
    elif scaling not in (None, "ntk"):
        raise NotImplementedError(f"rotary scaling {scaling!r}")
    return f.to(device) if device is not None else f, scale


def pack_mask(mask: torch.Tensor) -> torch.Tensor:
    """int32 [n, ceil(m / 32)] words of a bool mask [n, m]: bit j % 32 of word j // 32 of row i is
    mask[i, j] (the ``tree`` of :func:`paged_attention`)."""
    if mask.dim() != 2 or mask.dtype != torch.bool:
        raise ValueError("mask must be bool [n, m]")
    n, m = mask.shape
    words = max(1, -(-m // 32))
    bits = torch.zeros(n, words * 32, dtype=torch.int64, device=mask.device)
    bits[:, :m] = mask
    v = (bits.view(n, words, 32) << torch.arange(32, device=mask.device)).sum(-1)
    return torch.where(v >= 1 << 31, v - (1 << 32), v).to(torch.int32)


def tree_words(parents: Sequence[List[int]]) -> torch.Tensor:
    """``tree`` words (on the host) of several draft trees, one after the other: ``parents[b][i]`` is
    the parent of token i of sequence b, -1 for a child of the last verified token."""
    from .verify import tree_mask
    most = max((len(p) for p in parents), default=0)
    rows = []
    for p in parents:
        full = torch.zeros(len(p), max(most, 1), dtype=torch.bool)
        full[:, :len(p)] = tree_mask(p)
        rows.append(pack_mask(full))
    return torch.cat(rows) if rows else torch.zeros(0, 1, dtype=torch.int32)


def _cache(k: torch.Tensor, v: torch.Tensor, head_dim: int, dtype: torch.dtype, dev: torch.device):
    """The C description of a cache, checked."""
    if head_dim not in HEAD_DIMS:
        raise NotImplementedError(f"head_dim {head_dim} (supported: {HEAD_DIMS})")
    if k.dim() != 4 or k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype:
        raise ValueError("k_cache and v_cache must be [num_pages, kv_heads, page_size, row] of one dtype and "
                         "with the same strides")
    if k.device != dev or v.device != dev:
        raise ValueError("the cache must be on the device of the other tensors")
    pages, heads, size, row = k.shape
    if k.dtype == torch.uint8:
        bits, want, elem = 4, kv4_row_bytes(head_dim), 1
    elif k.dtype == dtype:
        bits, want, elem = 16, head_dim, 2
    else:
        raise ValueError(f"cache dtype {k.dtype} is neither {dtype} nor uint8 (4-bit)")
    if row != want:
        raise ValueError(f"a cache row must have {want} elements, got {row}")
    ps, hs, ts, es = k.stride()
    if es != 1 and row > 1:
        raise ValueError("a cache row must be contiguous")
    if size < 1 or size & (size - 1) or size > 65536:
        raise ValueError(f"page_size must be a power of two up to 65536, got {size}")
    if (ps * elem) % 16 or (hs * elem) % 16 or (ts * elem) % 16:
        raise ValueError("cache strides must be multiples of 16 bytes")
    return _native.PagedCache(k.data_ptr(), v.data_ptr(), pages, ps * elem, hs * elem, ts * elem, heads, size,
                              head_dim, bits)


def _rows(name: str, t: torch.Tensor, n: int, dtype: torch.dtype, dev: torch.device):
    """Checks [n, heads, head_dim] rows; strides of the first two dimensions are free."""
    if t.dim() != 3 or t.shape[0] != n:
        raise ValueError(f"{name} must be [{n}, heads, head_dim]")
    if t.dtype != dtype or t.device != dev:
        raise ValueError(f"{name} must have the dtype and device of q")
    ts, hs, es = t.stride()
    if es != 1 or ts % 8 or hs % 8:
        raise ValueError(f"{name}: head_dim must be contiguous and the other strides multiples of 8")
    return ts, hs


def _vector(name: str, t: torch.Tensor, dtype: torch.dtype, n: int, dev: torch.device):
    if t.dtype != dtype or t.dim() != 1 or t.numel() != n or t.device != dev or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous {dtype} [{n}] on the device of q")
    return t.data_ptr()


def _call(dev: torch.device, name: str, *args):
    """The library call on the tensors' device, whichever is current."""
    if torch.cuda.current_device() == dev.index:
        return _native.call(name, *args, _stream_ptr(dev))
    with torch.cuda.device(dev):
        return _native.call(name, *args, _stream_ptr(dev))


def _status_word(status: Optional[torch.Tensor], dev: torch.device):
    """(word to pass or None, whether to read it here): the caller's, or one of this call's own when
    ``SMB_DEBUG=1``."""
    if status is not None:
        if status.dtype != torch.int32 or status.numel() != 1 or status.device != dev:
            raise ValueError("status must be int32 [1] on the device of q")
        return status, False
    if ops.DEBUG:
        return torch.zeros(1, dtype=torch.int32, device=dev), True
    return None, False


#: Device code that ``status`` gets for a page or slot outside the cache.
BAD_PAGE = 2


def _raise_status(name: str, status: torch.Tensor):
    if int(status.item()) != 0:
        _native.check(name + " (device status)", -10 if int(status.item()) == BAD_PAGE else -9)


def kv_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
              slots: torch.Tensor, positions: Optional[torch.Tensor] = None,
              inv_freq: Optional[torch.Tensor] = None, *, interleaved: bool = False, rope_scale: float = 1.0,
              q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6,
              out: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotate the new tokens' queries and keys and write keys and values into the cache; returns the
    queries ``[N, Hq, head_dim]`` (``out``, contiguous, if given; it may not overlap q).

    q ``[N, Hq, head_dim]``, k and v ``[N, kv_heads, head_dim]`` (views of the projection's output are
    taken as they are).  ``slots`` int64 [N]: where each token goes; negative: nowhere.  The slots of
    a call have to be distinct.  ``positions`` int64 [N] and ``inv_freq`` float64 [rot / 2]
    (:func:`rope_inv_freq`) rotate the first ``rot`` dims: pairs (i, i + rot/2), or (2i, 2i + 1) when
    ``interleaved``; both None: no rotation.  ``q_norm`` / ``k_norm`` [head_dim]: weights of an RMS norm
    of each head before the rotation.  ``status`` int32 [1], set to :data:`BAD_PAGE` by a slot past
    the cache (which is not written)."""
    if not q.is_cuda:
        raise ValueError("q must be a CUDA tensor (no host path exists)")
    if q.dim() != 3:
        raise ValueError("q must be [N, heads, head_dim]")
    dev, dtype = q.device, q.dtype
    code = ops.storage_code(dtype)
    N, Hq, D = q.shape
    cache = _cache(k_cache, v_cache, D, dtype, dev)
    strides = (ctypes.c_int64 * 6)(*_rows("q", q, N, dtype, dev), *_rows("k", k, N, dtype, dev),
                                   *_rows("v", v, N, dtype, dev))
    if k.shape[1:] != (cache.kv_heads, D) or v.shape[1:] != (cache.kv_heads, D):
        raise ValueError(f"k and v must be [{N}, {cache.kv_heads}, {D}]")
    slots_p = _vector("slots", slots, torch.int64, N, dev)
    rot = pos_p = freq_p = 0
    if (positions is None) != (inv_freq is None):
        raise ValueError("positions and inv_freq go together")
    if inv_freq is not None:
        rot = 2 * inv_freq.numel()
        if rot % 16 or rot > D:
            raise ValueError(f"inv_freq must have a multiple of 8 entries, at most {D // 2}")
        pos_p = _vector("positions", positions, torch.int64, N, dev)
        freq_p = _vector("inv_freq", inv_freq, torch.float64, rot // 2, dev)
    qn_p = None if q_norm is None else _vector("q_norm", q_norm, dtype, D, dev)
    kn_p = None if k_norm is None else _vector("k_norm", k_norm, dtype, D, dev)
    if out is None:
        out = torch.empty(N, Hq, D, dtype=dtype, device=dev)
    elif out.shape != q.shape or out.dtype != dtype or out.device != dev or not out.is_contiguous():
        raise ValueError("out must be contiguous, with the shape, dtype and device of q")
    word, mine = _status_word(status, dev)
    _call(dev, "smb_kv_append", ctypes.byref(cache), q.data_ptr(), k.data_ptr(), v.data_ptr(), strides, code, N, Hq,
          slots_p, pos_p or None, freq_p or None, rot, int(interleaved), float(rope_scale), qn_p, kn_p, float(eps),
          out.data_ptr(), None if word is None else word.data_ptr())
    if mine:
        _raise_status("smb_kv_append", word)
    return out


def kv4_read(cache: torch.Tensor, slots: torch.Tensor, head_dim: int, dtype: torch.dtype,
             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values ``[M, kv_heads, head_dim]`` that the rows of ``slots`` (int64 [M]) of one array of a
    4-bit cache stand for.  A slot outside the cache reads as zeros."""
    if not cache.is_cuda:
        raise ValueError("cache must be a CUDA tensor (no host path exists)")
    if cache.dtype != torch.uint8:
        raise ValueError("cache must be a 4-bit cache (uint8)")
    dev = cache.device
    code = ops.storage_code(dtype)
    c = _cache(cache, cache, head_dim, dtype, dev)
    M = slots.numel()
    slots_p = _vector("slots", slots, torch.int64, M, dev)
    if out is None:
        out = torch.empty(M, c.kv_heads, head_dim, dtype=dtype, device=dev)
    elif out.shape != (M, c.kv_heads, head_dim) or out.dtype != dtype or out.device != dev or not out.is_contiguous():
        raise ValueError(f"out must be contiguous {dtype} [{M}, {c.kv_heads}, {head_dim}] on the cache's device")
    _call(dev, "smb_kv4_read", cache.data_ptr(), c.num_pages, c.kv_heads, c.page_size, head_dim, c.page_stride,
          c.head_stride, c.token_stride, code, slots_p, M, out.data_ptr())
    return out


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                    kv_lens: torch.Tensor, q_starts: torch.Tensor, *, tree: Optional[torch.Tensor] = None,
                    scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                    lse: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of each sequence's newest tokens over its cached keys and values -> [N, Hq, head_dim].

    Sequence b owns the rows ``q_starts[b]:q_starts[b + 1]`` of q ``[N, Hq, head_dim]`` (already appended
    to the cache) and ``kv_lens[b]`` keys, key j in page ``block_table[b, j // page_size]``.
    ``block_table`` int32 [B, max_pages], ``kv_lens`` int32 [B], ``q_starts`` int32 [B + 1].  Without
    ``tree`` the new tokens are causal.  ``tree`` int32 [N, words] (:func:`pack_mask`,
    :func:`tree_words`): token i sees every key before the sequence's new tokens, and new token t
    where bit t is set.  ``scale`` (positive) defaults to
    head_dim ** -0.5.  ``lse`` float32 [N, Hq], optional:
    receives the natural log of each softmax's sum (-inf, with an output of 0, for a token that sees no
    key).  Rows of q behind the last sequence leave ``out`` and ``lse`` as they were.  ``out`` may not
    overlap q.  ``status`` int32 [1] is set to :data:`BAD_PAGE` by a page outside the cache (its keys
    are left out)."""
    if not q.is_cuda:
        raise ValueError("q must be a CUDA tensor (no host path exists)")
    if q.dim() != 3:
        raise ValueError("q must be [N, heads, head_dim]")
    dev, dtype = q.device, q.dtype
    code = ops.storage_code(dtype)
    N, Hq, D = q.shape
    cache = _cache(k_cache, v_cache, D, dtype, dev)
    qts, qhs = _rows("q", q, N, dtype, dev)
    if Hq == 0 or Hq % cache.kv_heads:
        raise ValueError(f"{Hq} query heads are not a multiple of {cache.kv_heads} key heads")
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.device != dev:
        raise ValueError("block_table must be int32 [B, max_pages] on the device of q")
    B, max_pages = block_table.shape
    if max_pages > 1 and block_table.stride(1) != 1:
        raise ValueError("a row of block_table must be contiguous")
    lens_p = _vector("kv_lens", kv_lens, torch.int32, B, dev)
    starts_p = _vector("q_starts", q_starts, torch.int32, B + 1, dev)
    tree_p, tree_stride, words = None, 0, 0
    if tree is not None:
        if tree.dim() != 2 or tree.dtype != torch.int32 or tree.shape[0] != N or tree.device != dev:
            raise ValueError("tree must be int32 [N, words] on the device of q")
        words = tree.shape[1]
        if words < 1 or (words > 1 and tree.stride(1) != 1):
            raise ValueError("tree needs a word for each token, the words contiguous")
        tree_p, tree_stride = tree.data_ptr(), tree.stride(0)
    if out is None:
        out = torch.empty(N, Hq, D, dtype=dtype, device=dev)
    elif out.shape != q.shape:
        raise ValueError("out must have the shape of q")
    ots, ohs = _rows("out", out, N, dtype, dev)
    if lse is not None and (lse.dtype != torch.float32 or lse.shape != (N, Hq) or lse.device != dev
                            or not lse.is_contiguous()):
        raise ValueError("lse must be contiguous float32 [N, Hq] on the device of q")
    scale = float(D ** -0.5 if scale is None else scale)
    if not 0.0 < scale <= 1e30:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    word, mine = _status_word(status, dev)
    nbytes = _workspace_bytes(N, B, Hq, cache, dev)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _call(dev, "smb_paged_attention", ctypes.byref(cache), q.data_ptr(), qts, qhs, code, N, Hq, B,
          block_table.data_ptr(), block_table.stride(0) if B > 1 else max_pages, max_pages, lens_p, starts_p, tree_p,
          tree_stride, words, scale, out.data_ptr(), ots, ohs,
          None if lse is None else lse.data_ptr(), None if word is None else word.data_ptr(), ws.data_ptr(), nbytes)
    if mine:
        _raise_status("smb_paged_attention", word)
    return out


def _workspace_bytes(N: int, B: int, Hq: int, cache, dev: torch.device) -> int:
    fn = _native.load().smb_paged_attention_workspace_bytes
    if torch.cuda.current_device() == dev.index:
        n = fn(N, B, Hq, cache.kv_heads, cache.head_dim, cache.bits)
    else:
        with torch.cuda.device(dev):
            n = fn(N, B, Hq, cache.kv_heads, cache.head_dim, cache.bits)
    if n == 0:
        raise NotImplementedError(f"unsupported attention sizes N={N} B={B} Hq={Hq} kv_heads={cache.kv_heads} "
                                  f"head_dim={cache.head_dim}")
    return int(n)
