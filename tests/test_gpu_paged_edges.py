"""Paged cache and attention at the edges of the number formats (ae_b200/paged.py): non-finite values,
values of a 4-bit cache that overflow the 16-bit type, and weights below fp16's normal numbers.

A value of a 4-bit cache enters attention's second product as the 16-bit number nearest scale * code + zero.
Both numbers of a group can be finite and that one not (fp16: 15 * 4368 = 65520 rounds to infinity).  A row that may
not see such a value keeps its result bit for bit; a row that sees it gets that infinity (or NaN) in those
dims, and everywhere else the tolerance of ``tests/test_gpu_paged.py``, derived there."""
import math

import pytest
import torch

from tests import paged_reference as ref
from tests.test_gpu_paged import BF, FP, call, make_batch

pytestmark = pytest.mark.gpu

# Query heads over 2 key heads, 9 new tokens of 2 sequences: 5, 9, 18, 72 and 288 query rows of a key head on
# average, which go to the kernels for up to 8, 16 and 32 rows and to the tensor cores' with one and two row
# tiles at a time (heads of 256: to the first two).
HEADS = [2, 4, 8, 32, 128]
# scale and zero of a group as fractions of the largest finite number: code 15 overflows (in fp16 the scale that
# rounding gives the group 0 to 65504; bf16's rounding keeps that one finite), all but code 0, the negative side,
# and an infinite scale (code 0 is then NaN)
GROUPS = {"upper": (4368 / 65504, 0.0), "upper bf16": (0.0675, 0.0), "all": (4368 / 65504, 1.0),
          "lower": (-4368 / 65504, -0.5), "scale": (math.inf, 0.0)}


def masked_batch(heads, D, dtype, tree):
    """The batch of ``test_masked_places_may_hold_anything``; the rows that see the newest token but one of
    sequence 0."""
    d = make_batch([6, 3], [70, 35], heads, 2, D, 16, dtype, 4, tree, seed=11)
    if tree:
        d["tree"] = torch.tensor([1, 3, 5, 9, 17, 33, 1, 3, 7], dtype=torch.int32, device="cuda")[:, None].contiguous()
    return d, ([4] if tree else [4, 5])


def spoil(d, D, dtype, scale, zero):
    """Gives that token's values a second group of ``scale`` and ``zero`` with codes 0 to 15 in turn; returns its
    32 values as 16-bit numbers."""
    j = 70 - 2
    row = d["v_cache"][int(d["block_table"][0, j // 16]), :, j % 16]
    codes = torch.arange(32, device="cuda") % 16
    row[:, 16:32] = (codes[0::2] + 16 * codes[1::2]).to(torch.uint8)
    sz = torch.tensor([scale, zero], device="cuda", dtype=torch.float64).to(dtype)
    row[:, D // 2 + 4:D // 2 + 8] = sz.view(torch.uint8)
    return (codes.double() * sz[0].double() + sz[1].double()).to(dtype)


@pytest.mark.parametrize("tree", [False, True], ids=["causal", "tree"])
@pytest.mark.parametrize("dtype,kind", [(t, k) for t in (FP, BF) for k in GROUPS
                                        if k != ("upper bf16" if t == FP else "upper")])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("heads", HEADS)
def test_values_that_overflow_stay_behind_the_mask(heads, D, dtype, kind, tree):
    d, sees = masked_batch(heads, D, dtype, tree)
    good, good_lse = call(d)
    most = torch.finfo(dtype).max
    v16 = spoil(d, D, dtype, *(x * most for x in GROUPS[kind]))
    over = ~torch.isfinite(v16)
    assert bool(over.any()) and (kind == "scale") == bool(over.all())
    out, lse = call(d)
    assert torch.equal(lse, good_lse)  # keys are as they were
    for i in range(9):
        if i not in sees:
            assert torch.equal(out[i], good[i]), i
            continue
        got = out[i, :, 32:64]
        want = v16[over].double().expand(heads, -1)
        assert torch.equal(torch.nan_to_num(got[:, over].double(), nan=7.0), torch.nan_to_num(want, nan=7.0)), i
        assert torch.equal(out[i, :, :32], good[i, :, :32]) and torch.equal(out[i, :, 64:], good[i, :, 64:]), i
    if dtype == FP and kind in ("upper", "lower"):  # (sums of bf16's largest numbers pass 32 bits)
        # the finite neighbours in the group
        o, _, spread, reach = ref.attention(d["q"], d["k_cache"], d["v_cache"], d["block_table"], d["kv_lens"],
                                            d["q_starts"], d["tree"])
        u = ref.half_step(dtype)
        off = u * reach[..., None] if heads >= 32 and D <= 128 else torch.zeros_like(reach)[..., None]
        tol = u * o.abs() + (2 * u + 2 ** -14 + torch.expm1(2 * off)) * spread + 2 ** -25
        dims = 32 + torch.nonzero(~over)[:, 0]
        for i in sees:
            err = (out[i][:, dims].double() - o[i][:, dims]).abs()
            assert bool((err <= tol[i][:, dims]).all()), i


def append_values(v):
    """v [N, 1, D] appended as keys and as values of a 4-bit cache: both read back."""
    from ae_b200 import paged
    N, _, D = v.shape
    kc, vc = paged.new_cache(N // 16 + 1, 1, 16, D, v.dtype, "cuda", bits=4)
    slots = torch.arange(N, device="cuda")
    paged.kv_append(v.clone(), v, v, kc, vc, slots)
    return [paged.kv4_read(c, slots, D, v.dtype) for c in (kc, vc)]


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [FP, BF], ids=["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_nonfinite_values_are_not_lost_in_4_bits(D, dtype, value):
    """A NaN or an infinity among keys or values makes its group of 32 NaN, wherever in the group it is, and no other."""
    G = D // 32
    v = torch.randn(32 * G, 1, G, 32, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda").to(dtype)
    row = torch.arange(32 * G, device="cuda")
    want = torch.zeros(32 * G, 1, G, dtype=torch.bool, device="cuda")
    clean = append_values(v.view(-1, 1, D))
    v[row, 0, row // 32, row % 32] = value
    want[row, 0, row // 32] = True
    for got, was in zip(append_values(v.view(-1, 1, D)), clean):
        assert bool(torch.isnan(got.view_as(v)[want]).all())
        assert torch.equal(got.view_as(v)[~want], was.view_as(v)[~want])


@pytest.mark.parametrize("dtype", [FP, BF], ids=["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_values_that_fit_the_type_are_read_back_finite(D, dtype):
    """Groups that reach the largest finite number, from any smallest one (their span passes 32 bits in bf16).

    The scale is rounded to the type (u), or taken down to the largest one for which code 15 fits (2 u of the
    largest number less the zero, for code 15 to fall short), the zero is rounded (u |lo|), half a step for
    the code, and kv4_read rounds once (u |v|)."""
    most = torch.finfo(dtype).max
    g = torch.Generator(device="cuda").manual_seed(3)
    N = 512
    lo = torch.rand(N, 1, D // 32, 1, generator=g, device="cuda", dtype=torch.float64) * 2 - 1
    lo[::7] = -1.0
    lo[1::7] = 0.0
    hi = torch.ones_like(lo)
    hi[2::7] = 1 - 0.02 * torch.rand(hi[2::7].shape, generator=g, device="cuda", dtype=torch.float64)
    x = lo + (hi - lo) * torch.rand(N, 1, D // 32, 32, generator=g, device="cuda", dtype=torch.float64)
    x[..., 5:6], x[..., 9:10] = lo, hi
    v = (x * most).to(dtype)
    assert bool(torch.isfinite(v).all())
    v64 = v.double()
    lo, hi = v64.amin(-1, keepdim=True), v64.amax(-1, keepdim=True)
    u = ref.half_step(dtype)
    tol = (hi - lo) / 30 * (1 + 2 * u) + 2 * u * (most - lo) + u * lo.abs() + u * v64.abs()
    for got in append_values(v.view(N, 1, D)):
        assert bool(torch.isfinite(got).all())
        err = (got.double().view_as(v64) - v64).abs()
        assert bool((err <= tol * (1 + 2 ** -20)).all()), float((err / tol).max())


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("heads", [8, 32])
def test_nonfinite_values_in_every_masked_tile_again_and_again(heads, bits):
    """A tree of 300 tokens, two row tiles or more over the same masked tiles, in which each 13th token has NaN or
    infinite values and is seen by itself alone: the other rows are as they were, each time."""
    d = make_batch([300], [430], heads, 2, 128, 16, BF, bits, True, seed=12)
    bad = torch.arange(300, device="cuda") % 13 == 7
    words = d["tree"]
    for i in torch.nonzero(bad)[:, 0].tolist():
        bit = (1 << (i % 32)) - (1 << 32 if i % 32 == 31 else 0)
        words[:, i // 32] &= ~bit
        words[i, i // 32] |= bit
    good, good_lse = call(d)
    for i in torch.nonzero(bad)[:, 0].tolist():
        row = d["v_cache"][int(d["block_table"][0, (130 + i) // 16]), :, (130 + i) % 16]
        value = (math.nan, math.inf, -math.inf)[i % 3]
        if bits == 16:
            row[:] = value
        else:
            row[:, 64:80] = torch.tensor([1.0, value] * 4, dtype=BF, device="cuda").view(torch.uint8)
    for _ in range(30):
        out, lse = call(d)
        assert torch.equal(lse, good_lse) and torch.equal(out[~bad], good[~bad])
        assert not bool(torch.isfinite(out[bad]).any())


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [FP, BF], ids=["fp16", "bf16"])
@pytest.mark.parametrize("heads,D", [(2, 64), (16, 64), (32, 128), (32, 256), (64, 64), (64, 128), (256, 128)])
def test_many_small_weights_beside_large_ones(heads, D, dtype, bits):
    """Each 61st key has a weight of 1 and values of 0, the others weights of 2^-26 to 2^-20 and values of 30000, so
    that the output is theirs alone.

    fp16 has no 2^-26: a weight is kept at 2^7 of its size relative to the row's largest or more, and rounded to a
    multiple of 2^-24 there where it is below 2^-14: off by 2^-32 at most, of values of 30000, relative to the
    sum of the weights.  The rest as in ``tests/test_gpu_paged.py``."""
    N, n = 3000, 2
    d = make_batch([n], [N], heads, 2, D, 16, dtype, bits, False, seed=13)
    pages = d["k_cache"].shape[0]
    g = torch.Generator(device="cuda").manual_seed(14)
    k = torch.zeros(pages, 2, 16, D, dtype=torch.float64, device="cuda")
    v = torch.full_like(k, 30000.0)
    place = torch.zeros(pages * 16, dtype=torch.long, device="cuda")
    for b, p in enumerate(d["block_table"][0].tolist()):
        place[p * 16:p * 16 + 16] = torch.arange(b * 16, b * 16 + 16, device="cuda")
    large = (place.view(pages, 1, 16) % 61 == 0).expand(pages, 2, 16)
    k[..., 0] = torch.where(large, 0.0, -14 - 4 * torch.rand(pages, 2, 16, generator=g, device="cuda", dtype=torch.float64))
    v[large] = 0
    d["k_cache"], d["v_cache"] = ((ref.quantise(t, dtype)[0] if bits == 4 else t.to(dtype)) for t in (k, v))
    d["q"].zero_()
    d["q"][..., 0] = 1
    out, lse = call(d, scale=1.0)
    o, l, spread, reach = ref.attention(d["q"], d["k_cache"], d["v_cache"], d["block_table"], d["kv_lens"], d["q_starts"],
                                        scale=1.0)
    u = ref.half_step(dtype)
    off = u * reach if bits == 4 and heads > 32 and D <= 128 else torch.zeros_like(reach)
    lost = N * 2.0 ** -32 * 30000 / torch.exp(l) if dtype == FP else torch.zeros_like(l)  # (the largest score is 0)
    tol = u * o.abs() + (2 * u + 2 ** -14 + torch.expm1(2 * off)[..., None]) * spread + lost[..., None] + 2 ** -25
    err = (out.double() - o).abs()
    assert float(lost.max()) < 0.02 * float(o.abs().min())
    assert bool((err <= tol).all()), float((err / tol).max())
    assert bool(((lse.double() - l).abs() <= 2 ** -17 * (l.abs() + 8) + off).all())


@pytest.mark.parametrize("tree", [False, True], ids=["causal", "tree"])
@pytest.mark.parametrize("heads", HEADS)
def test_a_value_just_below_the_overflow_is_finite_in_every_kernel(heads, tree):
    """15 * 4368 - 2^-24 lies below the middle of 65504 and the next step, so the nearest fp16 is 65504 (rounded to 32
    bits first it would be the middle, and then infinite), also where another group of the token is not finite."""
    D = 128
    d, sees = masked_batch(heads, D, FP, tree)
    good, _ = call(d)
    spoil(d, D, FP, 4368.0, -2.0 ** -24)
    j = 70 - 2
    row = d["v_cache"][int(d["block_table"][0, j // 16]), :, j % 16]
    row[:, D // 2 + 12:D // 2 + 16] = torch.tensor([1.0, math.inf], device="cuda").to(FP).view(torch.uint8)
    out, _ = call(d)
    for i in range(9):
        if i not in sees:
            assert torch.equal(out[i], good[i]), i
        else:
            assert bool(torch.isfinite(out[i, :, :96]).all()) and bool(torch.isposinf(out[i, :, 96:]).all()), i
