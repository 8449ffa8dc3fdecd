"""Paged cache without a GPU: host helpers, the checks of the Python calls and of the C ABI."""
import ctypes
import math

import pytest
import torch

from ae_b200 import _native, build, paged


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _native.load()


def test_row_bytes(lib):
    for D, want in ((64, 48), (128, 80), (256, 160)):
        assert paged.kv4_row_bytes(D) == want == lib.smb_kv4_row_bytes(D)
    assert lib.smb_kv4_row_bytes(96) == -1
    with pytest.raises(NotImplementedError):
        paged.kv4_row_bytes(80)


def test_new_cache():
    k, v = paged.new_cache(3, 2, 16, 128, torch.bfloat16, "cpu")
    assert k.shape == v.shape == (3, 2, 16, 128) and k.dtype == torch.bfloat16 and int(k.count_nonzero()) == 0
    k, _ = paged.new_cache(3, 2, 16, 64, torch.float16, "cpu", bits=4)
    assert k.shape == (3, 2, 16, 48) and k.dtype == torch.uint8
    for bad in (dict(bits=8), dict(dtype=torch.float32), dict(head_dim=80)):
        args = dict(num_pages=1, kv_heads=1, page_size=16, head_dim=64, dtype=torch.float16, device="cpu")
        args.update(bad)
        with pytest.raises(NotImplementedError):
            paged.new_cache(**args)


def test_rope_frequencies():
    f, s = paged.rope_inv_freq(64, 10000.0)
    assert f.dtype == torch.float64 and s == 1.0 and f.shape == (32,)
    assert math.isclose(float(f[1]), 10000.0 ** (-2 / 64), rel_tol=1e-14)
    lin, _ = paged.rope_inv_freq(64, 10000.0, "linear", 4.0)
    assert torch.allclose(lin * 4, f, rtol=1e-15)
    ntk, _ = paged.rope_inv_freq(64, 10000.0, "ntk", 4.0)
    # the slowest pair turns exactly `factor` times slower, the fastest as before
    assert float(ntk[0]) == 1.0 and math.isclose(float(f[-1] / ntk[-1]), 4.0, rel_tol=1e-12)
    y, s = paged.rope_inv_freq(128, 1e4, "yarn", 8.0, trained=4096)
    g, _ = paged.rope_inv_freq(128, 1e4)
    ratio = g / y
    assert math.isclose(s, 0.1 * math.log(8.0) + 1.0)
    assert float(ratio[0]) == 1.0 and math.isclose(float(ratio[-1]), 8.0, rel_tol=1e-12)
    assert bool((ratio[1:] >= ratio[:-1] - 1e-12).all())
    turns = 4096 * g / (2 * math.pi)
    assert bool((ratio[turns > 40] < 1.2).all()) and bool((ratio[turns < 0.8] > 7.9).all())
    m, s = paged.rope_inv_freq(128, 5e5, "llama3", 8.0, trained=8192)
    g, _ = paged.rope_inv_freq(128, 5e5)
    turns = 8192 * g / (2 * math.pi)
    assert s == 1.0 and torch.equal(m[turns >= 4], g[turns >= 4])
    assert torch.allclose(m[turns <= 1] * 8, g[turns <= 1], rtol=1e-15)
    mid = (turns > 1) & (turns < 4)
    want = g * ((turns - 1) / 3) + g / 8 * (1 - (turns - 1) / 3)
    assert bool(mid.any()) and torch.allclose(m[mid], want[mid], rtol=1e-14)
    assert paged.rope_inv_freq(0)[0].shape == (0,)
    for bad in ((24, 1e4), (64, 1e4, "other"), (64, 1e4, "linear", 0.0)):
        with pytest.raises((ValueError, NotImplementedError)):
            paged.rope_inv_freq(*bad)


def test_pack_mask_and_tree_words():
    g = torch.Generator().manual_seed(0)
    mask = torch.rand(5, 70, generator=g) < 0.5
    w = paged.pack_mask(mask)
    assert w.shape == (5, 3) and w.dtype == torch.int32
    for i in range(5):
        for j in range(96):
            assert bool((int(w[i, j // 32]) >> (j % 32)) & 1) == (j < 70 and bool(mask[i, j]))
    assert paged.pack_mask(torch.zeros(2, 0, dtype=torch.bool)).shape == (2, 1)
    with pytest.raises(ValueError):
        paged.pack_mask(torch.zeros(2, 2))
    words = paged.tree_words([[-1, 0, 0, 2], [-1]])
    assert words.tolist() == [[1], [3], [5], [13], [1]]
    big = paged.tree_words([list(range(-1, 39)), [-1]])
    assert big.shape == (41, 2) and big[39].tolist() == [-1, 255] and big[40].tolist() == [1, 0]
    assert paged.tree_words([]).shape == (0, 1)


def test_cpu_tensors_are_refused(lib):
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    k = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    kc, vc = paged.new_cache(2, 2, 16, 64, torch.bfloat16, "cpu")
    i32 = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        paged.kv_append(q, k, k, kc, vc, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        paged.paged_attention(q, kc, vc, torch.zeros(2, 1, dtype=torch.int32), i32[:2], i32)
    with pytest.raises(ValueError, match="CUDA"):
        paged.kv4_read(kc.to(torch.uint8), torch.zeros(2, dtype=torch.int64), 64, torch.bfloat16)


class Cache(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("num_pages", ctypes.c_int64),
                ("page_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64), ("token_stride", ctypes.c_int64),
                ("kv_heads", ctypes.c_int), ("page_size", ctypes.c_int), ("head_dim", ctypes.c_int), ("bits", ctypes.c_int)]


class Append(ctypes.Structure):
    _fields_ = [("struct_bytes", ctypes.c_size_t), ("cache", Cache), ("q", ctypes.c_void_p), ("k", ctypes.c_void_p),
                ("v", ctypes.c_void_p), ("q_strides", ctypes.c_int64 * 2), ("k_strides", ctypes.c_int64 * 2),
                ("v_strides", ctypes.c_int64 * 2), ("slots", ctypes.c_void_p), ("positions", ctypes.c_void_p),
                ("inv_freq", ctypes.c_void_p), ("q_norm", ctypes.c_void_p), ("k_norm", ctypes.c_void_p),
                ("q_out", ctypes.c_void_p), ("status", ctypes.c_void_p), ("dtype", ctypes.c_int), ("N", ctypes.c_int),
                ("Hq", ctypes.c_int), ("rot", ctypes.c_int), ("interleaved", ctypes.c_int), ("rope_scale", ctypes.c_float),
                ("eps", ctypes.c_float)]


class Attention(ctypes.Structure):
    _fields_ = [("struct_bytes", ctypes.c_size_t), ("cache", Cache), ("q", ctypes.c_void_p),
                ("q_strides", ctypes.c_int64 * 2), ("out", ctypes.c_void_p), ("out_strides", ctypes.c_int64 * 2),
                ("block_table", ctypes.c_void_p), ("table_stride", ctypes.c_int64), ("kv_lens", ctypes.c_void_p),
                ("q_starts", ctypes.c_void_p), ("tree", ctypes.c_void_p), ("tree_stride", ctypes.c_int64),
                ("lse", ctypes.c_void_p), ("status", ctypes.c_void_p), ("ws", ctypes.c_void_p), ("ws_bytes", ctypes.c_size_t),
                ("dtype", ctypes.c_int), ("N", ctypes.c_int), ("Hq", ctypes.c_int), ("B", ctypes.c_int),
                ("max_pages", ctypes.c_int), ("tree_words", ctypes.c_int), ("scale", ctypes.c_float)]


def test_struct_formats_match_the_header():
    assert _native.CACHE_ARGS.size == ctypes.sizeof(Cache)
    assert _native.APPEND_ARGS.size == ctypes.sizeof(Append)
    assert _native.ATTENTION_ARGS.size == ctypes.sizeof(Attention)


def cache(**kw):
    d = dict(k=1024, v=2048, num_pages=4, page_stride=8192, head_stride=4096, token_stride=256, kv_heads=2, page_size=16,
             head_dim=128, bits=16)
    d.update(kw)
    return Cache(**d)


def status_of(fn, struct):
    return fn(ctypes.string_at(ctypes.addressof(struct), ctypes.sizeof(struct)), None)


SHAPE, DTYPE, ALIGN, NULL = -1, -2, -3, -8
BAD_CACHES = [(dict(bits=8), DTYPE), (dict(head_dim=96), SHAPE), (dict(page_size=24), SHAPE), (dict(page_size=0), SHAPE),
              (dict(page_size=1 << 17), SHAPE), (dict(kv_heads=0), SHAPE), (dict(num_pages=-1), SHAPE),
              (dict(token_stride=-256), SHAPE), (dict(token_stride=260), ALIGN), (dict(head_stride=8), ALIGN),
              (dict(page_stride=4), ALIGN), (dict(k=1028), ALIGN), (dict(v=8), ALIGN), (dict(k=None), NULL)]


@pytest.mark.parametrize("bad,code", BAD_CACHES)
def test_c_abi_refuses_bad_caches(lib, bad, code):
    a = Append(struct_bytes=ctypes.sizeof(Append), cache=cache(**bad), dtype=1, N=0, Hq=4)
    assert status_of(lib.smb_kv_append, a) == code
    b = Attention(struct_bytes=ctypes.sizeof(Attention), cache=cache(**bad), dtype=1, N=0, Hq=4, B=1, scale=1.0)
    assert status_of(lib.smb_paged_attention, b) == code


@pytest.mark.parametrize("bad,code", [
    (dict(struct_bytes=8), SHAPE), (dict(dtype=2), DTYPE), (dict(N=-1), SHAPE), (dict(Hq=0), SHAPE), (dict(Hq=2000), SHAPE),
    (dict(rot=24), SHAPE), (dict(rot=144), SHAPE), (dict(rot=-16), SHAPE), (dict(N=1), NULL),
    (dict(N=1, q=16, k=16, v=16, slots=16, q_out=16, rot=64), NULL),
    (dict(N=1, q=24, k=16, v=16, slots=16, q_out=16), ALIGN), (dict(N=1, q=16, k=16, v=16, slots=16, q_out=16), ALIGN), (dict(N=1, q=16, k=16, v=16, slots=16, q_out=16, k_norm=4), ALIGN),
    (dict(N=1, q=16, k=16, v=16, slots=16, q_out=16, k_strides=(ctypes.c_int64 * 2)(0, 4)), ALIGN), (dict(), 0)])
def test_c_abi_refuses_bad_appends(lib, bad, code):
    d = dict(struct_bytes=ctypes.sizeof(Append), cache=cache(), dtype=1, N=0, Hq=4)
    d.update(bad)
    assert status_of(lib.smb_kv_append, Append(**d)) == code


READY = dict(N=1, q=16, out=32, kv_lens=16, q_starts=16, ws=16, block_table=16, max_pages=1)


@pytest.mark.parametrize("bad,code", [
    (dict(struct_bytes=0), SHAPE), (dict(dtype=7), DTYPE), (dict(Hq=3), SHAPE), (dict(Hq=1), SHAPE), (dict(Hq=2048), SHAPE),
    (dict(B=-1), SHAPE), (dict(N=1 << 30), SHAPE), (dict(scale=0.0), SHAPE), (dict(scale=-1.0), SHAPE),
    (dict(scale=float("nan")), SHAPE), (dict(scale=float("inf")), SHAPE), (dict(max_pages=-1), SHAPE),
    (dict(tree=16, tree_words=0), SHAPE), (dict(N=1), NULL), (dict(READY, block_table=None), NULL), (dict(READY, ws=None), NULL),
    (dict(READY, cache=cache(num_pages=0)), SHAPE), (dict(READY, out=16), ALIGN), (dict(READY, q=8), ALIGN), (dict(READY, out=4), ALIGN), (dict(READY, q_strides=(ctypes.c_int64 * 2)(128, 20)), ALIGN),
    (dict(B=0, N=1), 0), (dict(), 0)])
def test_c_abi_refuses_bad_attention(lib, bad, code):
    d = dict(struct_bytes=ctypes.sizeof(Attention), cache=cache(), dtype=1, N=0, Hq=4, B=1, scale=1.0)
    d.update(bad)
    assert status_of(lib.smb_paged_attention, Attention(**d)) == code


@pytest.mark.parametrize("page_size,most", [(1, 1 << 30), (16, 1 << 26), (65536, 1 << 14)])
def test_c_abi_refuses_tables_of_more_than_30_bits(lib, page_size, most):
    """Key indexes, and the end of the tile behind the last key, are 32-bit integers."""
    d = dict(struct_bytes=ctypes.sizeof(Attention), cache=cache(page_size=page_size), dtype=1, N=0, Hq=4, B=1, scale=1.0)
    assert status_of(lib.smb_paged_attention, Attention(**d, max_pages=most)) == 0
    assert status_of(lib.smb_paged_attention, Attention(**d, max_pages=most + 1)) == SHAPE
    assert status_of(lib.smb_paged_attention, Attention(**d, max_pages=(1 << 31) - 1)) == SHAPE


def test_c_abi_null_and_read(lib):
    assert lib.smb_kv_append(None, None) == NULL and lib.smb_paged_attention(None, None) == NULL
    assert lib.smb_kv4_read(None, 1, None, 1, None, None) == NULL

    def read(c, *args):
        return lib.smb_kv4_read(ctypes.string_at(ctypes.addressof(c), ctypes.sizeof(c)), *args)

    assert read(cache(), 1, None, 0, None, None) == DTYPE             # not a 4-bit cache
    c4 = cache(bits=4)
    assert read(c4, 9, None, 0, None, None) == DTYPE
    assert read(c4, 1, None, -1, None, None) == SHAPE
    assert read(c4, 1, None, 0, None, None) == 0
    assert read(c4, 1, None, 3, None, None) == NULL
    assert read(c4, 1, 16, 3, 20, None) == ALIGN
    for sizes in ((1, 1, 3, 2, 128, 16), (1, 1, 4, 2, 100, 16), (1, 1, 4, 2, 128, 8), (-1, 1, 4, 2, 128, 16)):
        assert lib.smb_paged_attention_workspace_bytes(*sizes) == 0


def test_verify_decoder_names_its_caches():
    from ae_b200.verify import DecoderConfig, VerifyDecoder
    cfg = DecoderConfig(layers=1, H=64, I=64, E=2, k=1, heads=2, kv_heads=1, head_dim=64, vocab=10)
    with pytest.raises(ValueError, match="cache"):
        VerifyDecoder(cfg, 1, 2, 2, "cpu", cache="other")
