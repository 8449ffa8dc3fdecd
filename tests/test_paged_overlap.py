"""Outputs of the paged cache's calls that overlap their inputs are refused (ae_b200/paged.py): the test of
two sets of rows against sets of addresses (CPU), and the calls' refusals (GPU; nothing is launched)."""
import random

import pytest
import torch

from ae_b200 import paged


def view(buf, n, h, D, ts, hs, at):
    return buf.as_strided((n, h, D), (ts, hs, 1), at)


def addresses(t):
    return {t.storage_offset() + i * t.stride(0) + j * t.stride(1) + d
            for i in range(t.shape[0]) for j in range(t.shape[1]) for d in range(t.shape[2])}


def test_rows_that_share_elements():
    rng = random.Random(0)
    buf = torch.zeros(4096, dtype=torch.bfloat16)
    seen = {True: 0, False: 0}
    for _ in range(3000):
        D = 8
        ta = (rng.randint(1, 4), rng.randint(1, 4), D, 8 * rng.randint(0, 12), 8 * rng.randint(0, 12))
        tb = (rng.randint(1, 4), rng.randint(1, 4), D, *(ta[3:] if rng.random() < 0.5 else
                                                        (8 * rng.randint(0, 12), 8 * rng.randint(0, 12))))
        a, b = view(buf, *ta, rng.randint(0, 300)), view(buf, *tb, rng.randint(0, 300))
        want = bool(addresses(a) & addresses(b))
        assert paged._overlap(a, b) == want == paged._overlap(b, a), (ta, tb)
        seen[want] += 1
    assert min(seen.values()) > 500


def test_slices_of_one_buffer_do_not_overlap():
    x = torch.zeros(70, 12, 64, dtype=torch.float16)
    assert not paged._overlap(x[:, :6], x[:, 6:]) and not paged._overlap(x[:35], x[35:])
    assert paged._overlap(x[:, :7], x[:, 6:]) and paged._overlap(x[:36], x[35:])
    y = x.transpose(0, 1)  # heads outside
    assert not paged._overlap(y[:6], y[6:]) and not paged._overlap(y[:, :35], y[:, 35:])
    assert not paged._overlap(x[::2], x[1::2]) and not paged._overlap(x[:, ::2], x[:, 1::2])
    assert not paged._overlap(x[:0], x) and not paged._overlap(x, x.clone()) and paged._overlap(x, x)


@pytest.mark.gpu
def test_attention_refuses_an_out_over_q():
    from tests.test_gpu_paged import make_batch
    d = make_batch([3, 1], [40, 7], 4, 2, 128, 16, torch.bfloat16, 16, False)
    want = paged.paged_attention(**d)
    buf = torch.zeros(16, 4, 128, dtype=torch.bfloat16, device="cuda")
    buf[8:12] = d["q"]
    d["q"] = buf[8:12]
    for out in (buf[8:12], buf[7:11], buf[11:15], buf.view(-1)[7 * 512 + 64:11 * 512 + 64].view(4, 4, 128)):
        with pytest.raises(ValueError, match="overlap q"):
            paged.paged_attention(**d, out=out)
    for out in (buf[4:8], buf[12:16]):
        assert torch.equal(paged.paged_attention(**d, out=out), want)


@pytest.mark.gpu
def test_append_refuses_an_out_over_its_inputs_and_one_array_for_both():
    x = torch.randn(4, 8, 64, generator=torch.Generator(device="cuda").manual_seed(0), device="cuda").to(torch.float16)
    kc, vc = paged.new_cache(2, 2, 16, 64, torch.float16, "cuda")
    slots = torch.arange(4, device="cuda")
    q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
    buf = torch.zeros(1536, dtype=torch.float16, device="cuda")
    out, over = buf[512:].view(4, 4, 64), buf[256:768].view(4, 2, 64)
    flat = x.view(-1)
    for name, args, o in (("q", (q, k, v), flat[:1024].view(4, 4, 64)), ("q", (q, k, v), flat[1024:].view(4, 4, 64)),
                          ("k", (q, over, v), out), ("v", (q, k, over), out)):
        with pytest.raises(ValueError, match=f"overlap {name}"):
            paged.kv_append(*args, kc, vc, slots, out=o)
    with pytest.raises(ValueError, match="same array"):
        paged.kv_append(q, k, v, kc, kc, slots)
    assert torch.equal(paged.kv_append(q, k, v, kc, vc, slots, out=out), q)


def test_rows_of_a_cache_that_run_into_one_another():
    def f(levels, row):
        (ps, pages), (hs, heads), (ts, size) = levels
        return paged._cache_rows_overlap((pages, ps, hs, ts, heads, size), row)

    assert not f(((8192, 4), (4096, 2), (256, 16)), 256)           # heads outside tokens
    assert not f(((8192, 4), (256, 2), (512, 16)), 256)            # tokens outside heads, a token-major pool
    assert not f(((65536, 4), (256, 2), (768, 16)), 256)           # a slice of its heads
    assert not f(((0, 1), (0, 1), (80, 16)), 80) and not f(((5, 1), (7, 1), (3, 1)), 256)
    for bad in (((8192, 4), (0, 2), (256, 16)), ((0, 4), (4096, 2), (256, 16)), ((8192, 4), (4096, 2), (240, 16)),
                ((8176, 4), (4096, 2), (256, 16)), ((8192, 4), (256, 2), (256, 16))):
        assert f(bad, 256), bad


@pytest.mark.gpu
def test_append_refuses_a_cache_of_repeated_rows():
    x = torch.zeros(4, 8, 64, dtype=torch.float16, device="cuda")
    kc, vc = (t[:, :1].expand(2, 2, 16, 64) for t in paged.new_cache(2, 1, 16, 64, torch.float16, "cuda"))
    slots = torch.arange(4, device="cuda")
    with pytest.raises(ValueError, match="rows of a cache"):
        paged.kv_append(x[:, :4], x[:, 4:6], x[:, 6:], kc, vc, slots)
    i32 = dict(dtype=torch.int32, device="cuda")
    out = paged.paged_attention(x[:1, :4].contiguous(), kc, vc, torch.zeros(1, 1, **i32), torch.ones(1, **i32),
                                torch.tensor([0, 1], **i32))       # (read, it may be)
    assert bool((out == 0).all())
