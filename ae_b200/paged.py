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

import functools
import math
from typing import List, Optional, Sequence, Tuple

import numpy as np
import torch

from . import _native, ops

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


def _cache(k: torch.Tensor, v: torch.Tensor, head_dim: int, dtype: torch.dtype, dev: int):
    """The fields of the C description of a cache (``smb_paged_cache_t``), checked."""
    if head_dim not in HEAD_DIMS:
        raise NotImplementedError(f"head_dim {head_dim} (supported: {HEAD_DIMS})")
    shape, stride, kind = k.shape, k.stride(), k.dtype
    if len(shape) != 4 or v.shape != shape or v.stride() != stride or v.dtype != kind:
        raise ValueError("k_cache and v_cache must be [num_pages, kv_heads, page_size, row] of one dtype and "
                         "with the same strides")
    if k.get_device() != dev or v.get_device() != dev:
        raise ValueError("the cache must be on the device of the other tensors")
    pages, heads, size, row = shape
    ps, hs, ts, es = stride
    if kind == dtype:
        bits, want = 16, head_dim
        ps, hs, ts = 2 * ps, 2 * hs, 2 * ts
    elif kind == torch.uint8:
        bits, want = 4, kv4_row_bytes(head_dim)
    else:
        raise ValueError(f"cache dtype {kind} is neither {dtype} nor uint8 (4-bit)")
    if row != want:
        raise ValueError(f"a cache row must have {want} elements, got {row}")
    if es != 1:
        raise ValueError("a cache row must be contiguous")
    if heads < 1 or size < 1 or size & (size - 1) or size > 65536:
        raise ValueError(f"page_size must be a power of two up to 65536, got {size}")
    if (ps | hs | ts) & 15:
        raise ValueError("cache strides must be multiples of 16 bytes")
    return k.data_ptr(), v.data_ptr(), pages, ps, hs, ts, heads, size, head_dim, bits


@functools.lru_cache(maxsize=1024)
def _cache_rows_overlap(sizes, row: int) -> bool:
    """Whether rows of ``row`` bytes run into one another; ``sizes``: (pages, page stride, head stride, token stride,
    heads, page size), strides in bytes."""
    pages, ps, hs, ts, heads, size = sizes
    end = row
    for stride, n in sorted(((ps, pages), (hs, heads), (ts, size))):
        if n > 1:
            if stride < end:
                return True
            end += stride * (n - 1)
    return False


def _rows(name: str, t: torch.Tensor, shape, dtype: torch.dtype, dev: int):
    """Checks [n, heads, head_dim] rows (the first two strides are free); returns those strides."""
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    if t.dtype != dtype or t.get_device() != dev:
        raise ValueError(f"{name} must have the dtype and device of q")
    ts, hs, es = t.stride()
    if es != 1 or (ts | hs) & 7:
        raise ValueError(f"{name}: head_dim must be contiguous and the other strides multiples of 8")
    return ts, hs


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two sets of rows [n, heads, head_dim] (rows contiguous, one dtype) share an element."""
    D = a.shape[2]
    if a.numel() == 0 or b.numel() == 0:
        return False
    levels = [sorted(((s, n) for s, n in zip(t.stride(), t.shape[:2]) if n > 1), reverse=True) for t in (a, b)]
    pa, pb = (t.data_ptr() // t.element_size() for t in (a, b))

    def span(lv):
        return sum(s * (n - 1) for s, n in lv) + D

    if pa + span(levels[0]) <= pb or pb + span(levels[1]) <= pa:
        return False
    if levels[0] and levels[1] and levels[0][0][0] == levels[1][0][0] > 0:
        # slices of one buffer: side by side within its outer stride
        period, ea, eb = levels[0][0][0], span(levels[0][1:]), span(levels[1][1:])
        if ea <= (pb - pa) % period <= period - eb:
            return False
    starts = [np.sort(np.add.outer(np.arange(t.shape[0]) * t.stride(0), np.arange(t.shape[1]) * t.stride(1)).ravel() + p)
              for t, p in ((a, pa), (b, pb))]
    after = np.searchsorted(starts[1], starts[0] - D, side="right")  # the first row of b that ends behind a's start
    near = after < starts[1].size
    return bool((starts[1][after[near]] < starts[0][near] + D).any())


def _vector(name: str, t: torch.Tensor, dtype: torch.dtype, n: int, dev: int) -> int:
    if t.dtype != dtype or t.shape != (n,) or t.get_device() != dev or (n > 1 and t.stride(0) != 1):
        raise ValueError(f"{name} must be contiguous {dtype} [{n}] on the device of q")
    return t.data_ptr()


def _launch(dev: int, fn, *args):
    """The library call on the tensors' device, whichever is current, and its current stream."""
    if torch._C._cuda_getDevice() == dev:
        return fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    with torch.cuda.device(dev):
        return fn(*args, torch._C._cuda_getCurrentRawStream(dev))


def _status_word(status: Optional[torch.Tensor], dev: int):
    """(word to pass or None, whether to read it here): the caller's, or one of this call's own when
    ``SMB_DEBUG=1``."""
    if status is not None:
        if status.dtype != torch.int32 or status.numel() != 1 or status.get_device() != dev:
            raise ValueError("status must be int32 [1] on the device of q")
        return status, False
    if ops.DEBUG:
        return torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", dev)), True
    return None, False


#: Device codes that ``status`` gets (the first one stays): a page or slot outside the cache, which was left
#: out, and a device wait of :func:`paged_attention` that ran past its limit, after which the call's results are
#: void.  Without a ``status`` of the caller's, and without ``SMB_DEBUG=1``, neither is recorded anywhere.
BAD_PAGE = 2
TIMEOUT = 1


def _raise_status(name: str, status: torch.Tensor):
    code = int(status.item())
    if code != 0:
        _native.check(name + " (device status)", -10 if code == BAD_PAGE else -9)


def check_status(status: torch.Tensor):
    """Reads (synchronously) and clears the ``status`` word of earlier calls; raises what it holds."""
    try:
        _raise_status("paged cache", status)
    except _native.NativeError:
        status.zero_()
        raise


def _query(q: torch.Tensor):
    if not q.is_cuda:
        raise ValueError("q must be a CUDA tensor (no host path exists)")
    shape = q.shape
    if len(shape) != 3 or shape[1] < 1:
        raise ValueError("q must be [N, heads, head_dim]")
    return q.get_device(), q.dtype, ops.storage_code(q.dtype), shape


def kv_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
              slots: torch.Tensor, positions: Optional[torch.Tensor] = None,
              inv_freq: Optional[torch.Tensor] = None, *, interleaved: bool = False, rope_scale: float = 1.0,
              q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6,
              out: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotate the new tokens' queries and keys and write keys and values into the cache; returns the
    queries ``[N, Hq, head_dim]`` (``out``, contiguous, if given; it may not overlap q, k or v).

    q ``[N, Hq, head_dim]``, k and v ``[N, kv_heads, head_dim]`` (views of the projection's output are
    taken as they are).  ``slots`` int64 [N]: where each token goes; negative: nowhere.  The slots of
    a call, and the rows of the cache, have to be distinct.  ``positions`` int64 [N] and ``inv_freq`` float64 [rot / 2]
    (:func:`rope_inv_freq`) rotate the first ``rot`` dims: pairs (i, i + rot/2), or (2i, 2i + 1) when
    ``interleaved``; both None: no rotation.  ``q_norm`` / ``k_norm`` [head_dim]: weights of an RMS norm
    of each head before the rotation.  Values that fit the type stay finite in a 4-bit cache; a group
    of 32 dims with a NaN or an infinity among them reads as NaN.  ``status`` int32 [1], set to
    :data:`BAD_PAGE` by a slot past the cache (which is not written)."""
    dev, dtype, code, shape = _query(q)
    N, Hq, D = shape
    cache = _cache(k_cache, v_cache, D, dtype, dev)
    kv_shape = (N, cache[6], D)
    strides = _rows("q", q, shape, dtype, dev) + _rows("k", k, kv_shape, dtype, dev) + _rows("v", v, kv_shape, dtype, dev)
    slots_p = _vector("slots", slots, torch.int64, N, dev)
    rot = pos_p = freq_p = 0
    if (positions is None) != (inv_freq is None):
        raise ValueError("positions and inv_freq go together")
    if inv_freq is not None:
        rot = 2 * inv_freq.numel()
        if rot & 15 or rot > D:
            raise ValueError(f"inv_freq must have a multiple of 8 entries, at most {D // 2}")
        pos_p = _vector("positions", positions, torch.int64, N, dev)
        freq_p = _vector("inv_freq", inv_freq, torch.float64, rot // 2, dev)
    qn_p = 0 if q_norm is None else _vector("q_norm", q_norm, dtype, D, dev)
    kn_p = 0 if k_norm is None else _vector("k_norm", k_norm, dtype, D, dev)
    if out is None:
        out = q.new_empty(shape)
    elif out.shape != shape or out.dtype != dtype or out.get_device() != dev or not out.is_contiguous():
        raise ValueError("out must be contiguous, with the shape, dtype and device of q")
    else:
        for name, t in (("q", q), ("k", k), ("v", v)):
            if _overlap(out, t):
                raise ValueError(f"out may not overlap {name}")
    if N > 0 and cache[2] > 0:
        if cache[0] == cache[1]:
            raise ValueError("k_cache and v_cache may not be the same array")
        if _cache_rows_overlap(cache[2:8], 2 * D if cache[9] == 16 else kv4_row_bytes(D)):
            raise ValueError("the rows of a cache to append to may not overlap")
    word, mine = _status_word(status, dev)
    args = _native.APPEND_ARGS
    rc = _launch(dev, _native.load().smb_kv_append, args.pack(
        args.size, *cache, q.data_ptr(), k.data_ptr(), v.data_ptr(), *strides, slots_p, pos_p, freq_p, qn_p, kn_p,
        out.data_ptr(), 0 if word is None else word.data_ptr(), code, N, Hq, rot, bool(interleaved), rope_scale, eps))
    if rc:
        _native.check("smb_kv_append", rc)
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
    dev = cache.get_device()
    code = ops.storage_code(dtype)
    c = _cache(cache, cache, head_dim, dtype, dev)
    M = slots.numel()
    slots_p = _vector("slots", slots, torch.int64, M, dev)
    shape = (M, c[6], head_dim)
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=cache.device)
    elif out.shape != shape or out.dtype != dtype or out.get_device() != dev or not out.is_contiguous():
        raise ValueError(f"out must be contiguous {dtype} {list(shape)} on the cache's device")
    rc = _launch(dev, _native.load().smb_kv4_read, _native.CACHE_ARGS.pack(*c), code, slots_p, M, out.data_ptr())
    if rc:
        _native.check("smb_kv4_read", rc)
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
    where bit t is set.  ``scale`` (positive) defaults to head_dim ** -0.5.  ``lse`` float32 [N, Hq],
    optional: receives the natural log of each softmax's sum (-inf, with an output of 0, for a token
    that sees no key).  Rows of q behind the last sequence leave ``out`` and ``lse`` as they were.
    ``out`` may not overlap q.  ``status`` int32 [1] is set to :data:`BAD_PAGE` by a page outside the
    cache (its keys are left out), to :data:`TIMEOUT` by a call whose results are void;
    :func:`check_status` reads it."""
    dev, dtype, code, shape = _query(q)
    N, Hq, D = shape
    cache = _cache(k_cache, v_cache, D, dtype, dev)
    qts, qhs = _rows("q", q, shape, dtype, dev)
    if Hq % cache[6]:
        raise ValueError(f"{Hq} query heads are not a multiple of {cache[6]} key heads")
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.get_device() != dev:
        raise ValueError("block_table must be int32 [B, max_pages] on the device of q")
    B, max_pages = block_table.shape
    if max_pages * cache[7] > 1 << 30:
        raise ValueError(f"block_table has {max_pages} pages of {cache[7]} tokens for a sequence (at most 2^30 tokens)")
    table_stride, one = block_table.stride()
    if max_pages > 1 and one != 1:
        raise ValueError("a row of block_table must be contiguous")
    lens_p = _vector("kv_lens", kv_lens, torch.int32, B, dev)
    starts_p = _vector("q_starts", q_starts, torch.int32, B + 1, dev)
    tree_p = tree_stride = words = 0
    if tree is not None:
        if tree.dim() != 2 or tree.dtype != torch.int32 or tree.shape[0] != N or tree.get_device() != dev:
            raise ValueError("tree must be int32 [N, words] on the device of q")
        words = tree.shape[1]
        tree_stride, one = tree.stride()
        if words < 1 or (words > 1 and one != 1):
            raise ValueError("tree needs a word for each token, the words contiguous")
        tree_p = tree.data_ptr()
        if N == 0:
            tree_p = 0
    given = out is not None
    if not given:
        out = q.new_empty(shape)
    ots, ohs = _rows("out", out, shape, dtype, dev)
    (inner, n), (outer, m) = sorted(((ots, N), (ohs, Hq)))
    if (n > 1 and inner < D) or (m > 1 and outer < inner * (n - 1) + D):
        raise ValueError("the rows of out may not overlap")
    if given and _overlap(out, q):
        raise ValueError("out may not overlap q")
    if N > 0 and B > 0 and cache[2] == 0:
        raise ValueError("the cache has no pages")
    if lse is not None and (lse.dtype != torch.float32 or lse.shape != (N, Hq) or lse.get_device() != dev
                            or not lse.is_contiguous()):
        raise ValueError("lse must be contiguous float32 [N, Hq] on the device of q")
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale <= 1e30:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    word, mine = _status_word(status, dev)
    nbytes = _workspace_bytes(N, B, Hq, cache[6], D, cache[9], dev)
    ws = q.new_empty(nbytes >> 1)  # 16-bit elements
    args = _native.ATTENTION_ARGS
    rc = _launch(dev, _native.load().smb_paged_attention, args.pack(
        args.size, *cache, q.data_ptr(), qts, qhs, out.data_ptr(), ots, ohs, block_table.data_ptr(), table_stride,
        lens_p, starts_p, tree_p, tree_stride, 0 if lse is None else lse.data_ptr(),
        0 if word is None else word.data_ptr(), ws.data_ptr(), nbytes, code, N, Hq, B, max_pages, words, scale))
    if rc:
        _native.check("smb_paged_attention", rc)
    if mine:
        _raise_status("smb_paged_attention", word)
    return out


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(N: int, B: int, Hq: int, Hkv: int, D: int, bits: int, dev: int) -> int:
    with torch.cuda.device(dev):
        n = _native.load().smb_paged_attention_workspace_bytes(N, B, Hq, Hkv, D, bits)
    if n == 0:
        raise NotImplementedError(f"unsupported attention sizes N={N} B={B} Hq={Hq} kv_heads={Hkv} head_dim={D}")
    return int(n)
