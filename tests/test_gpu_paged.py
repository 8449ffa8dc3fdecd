"""Paged key/value cache on the GPU (ae_b200/paged.py): append and attention against plain 64-bit
forms.

Tolerances, per element, u = half a step of the 16-bit type (2^-8 bf16, 2^-11 fp16):
* append: one rounding, u |y|, of a value whose 32-bit error is a few 2^-24 of the terms it is made
  of (norm, two products, angle of 2^-23 turns): + 2^-18 of the head's largest value.
* attention: the weights p are rounded once (u, relative to sum p |v|), the output once (u |y|), the
  values of a 4-bit cache once more (u sum p |v|); scores and exponentials in 32 bits: 2^-14 of
  sum p |v|.
* lse: 32-bit scores of size up to 40: 2^-17 (|lse| + 8).
* many query rows over a 4-bit cache (more than 32 rows of a key head on average, head sizes 64 and
  128): the keys' values are rounded to the 16-bit type, each by u of itself at most, so a score is
  off by d = u scale sum |q k| at most, lse by d, a weight p by a factor within e^(+-2d): e^(2d) - 1
  of sum p |v|."""
import math

import pytest
import torch

from tests import paged_reference as ref

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make_cache(g, pages, Hkv, ps, D, dtype, bits):
    x = torch.randn(pages, Hkv, ps, D, generator=g, device="cuda", dtype=torch.float64)
    return ref.quantise(x, dtype)[0] if bits == 4 else x.to(dtype)


def make_batch(new, keys, Hq, Hkv, D, ps, dtype, bits, tree, seed=0, spare=2, words=None):
    g = gen(seed)
    used = [-(-max(k, 1) // ps) for k in keys]
    pages = sum(used) + spare
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(new), max(used)), 1 << 30, dtype=torch.int32, device="cuda")  # past the used: never read
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = order[at:at + u]
        at += u
    N = sum(new)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    d = dict(q=torch.randn(N, Hq, D, generator=g, device="cuda").mul_(1.5).to(dtype),
             k_cache=make_cache(g, pages, Hkv, ps, D, dtype, bits), v_cache=make_cache(g, pages, Hkv, ps, D, dtype, bits),
             block_table=table, kv_lens=torch.tensor(keys, dtype=torch.int32, device="cuda"),
             q_starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), tree=None)
    if tree:
        words = words or -(-max(new) // 32)
        d["tree"] = torch.randint(-(1 << 31), (1 << 31) - 1, (N, words), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
    return d


def call(d, **kw):
    from ae_b200 import paged
    lse = torch.full(d["q"].shape[:2], 7.0, dtype=torch.float32, device="cuda")
    out = torch.full_like(d["q"], 7.0, memory_format=torch.contiguous_format)
    paged.paged_attention(d["q"], d["k_cache"], d["v_cache"], d["block_table"], d["kv_lens"], d["q_starts"],
                          tree=d["tree"], out=out, lse=lse, **kw)
    return out, lse


def compare(d, out, lse, **kw):
    table = d["block_table"]
    o, l, spread, reach = ref.attention(d["q"], d["k_cache"], d["v_cache"], table, d["kv_lens"], d["q_starts"], d["tree"], **kw)
    own = ~torch.isnan(l)
    u = ref.half_step(d["q"].dtype)
    more = 1 if d["k_cache"].dtype == torch.uint8 else 0
    tol = u * o.abs() + ((1 + more) * u + 2 ** -14) * spread + 2 ** -25
    Hkv, D = d["k_cache"].shape[1], d["q"].shape[2]
    rows = -(-d["q"].shape[0] * (d["q"].shape[1] // Hkv) // table.shape[0])
    off = torch.zeros_like(reach)
    if more and rows > 32 and D <= 128:
        off = u * reach
        tol = tol + torch.expm1(2 * off)[..., None] * spread
    err = (out.double() - o).abs()
    assert bool((err[own] <= tol[own]).all()), float((err - tol)[own].max())
    assert bool((out[~own] == 7.0).all()) and bool((lse[~own] == 7.0).all())
    assert torch.equal(torch.isinf(lse[own]), torch.isinf(l[own]))
    fin = own & torch.isfinite(l)
    assert bool(((lse.double() - l).abs()[fin] <= (2 ** -17 * (l.abs() + 8) + off)[fin]).all())


SHAPES = [
    # new, keys, Hq, Hkv, D, ps, tree
    ([1], [1], 1, 1, 64, 1, False),
    ([1, 1, 1], [1, 63, 64], 4, 2, 128, 16, False),
    ([1, 1], [65, 1000], 8, 8, 128, 32, False),
    ([1, 1, 1, 1], [0, 5, 700, 2049], 8, 2, 256, 16, False),
    ([1], [5000], 32, 1, 64, 64, False),
    ([1, 1], [300, 17], 70, 2, 128, 8, False),         # 35 heads on one key head: more than a row tile
    ([7, 1, 30], [7, 900, 31], 5, 1, 128, 2, False),   # 5 heads: row tiles that do not divide
    ([33, 0, 2], [200, 10, 2], 8, 4, 64, 128, False),
    ([150], [400], 8, 4, 128, 16, False),
    ([40, 3], [20, 1], 4, 2, 128, 16, False),          # fewer keys than new tokens: rows that see nothing
    ([32, 32], [97, 1032], 32, 8, 128, 64, True),
    ([20, 64, 1], [20, 64, 130], 12, 2, 64, 16, True),
    ([33, 5], [170, 2], 3, 3, 256, 32, True),
    ([70, 100], [333, 100], 6, 1, 128, 16, True),
    # many rows: one and two row tiles of 128 at a time, short and long, pages from 8 to 256
    ([16, 40, 9], [16, 3000, 500], 8, 2, 64, 8, True),
    ([64], [5000], 4, 2, 128, 256, False),
    ([60, 3, 64], [60, 130, 127], 6, 3, 128, 128, False),
    ([300, 500, 0, 7], [1300, 500, 3, 260], 16, 8, 64, 32, False),
    ([33] * 40, [33 + 29 * i for i in range(40)], 8, 2, 128, 64, True),
    ([200], [100], 10, 2, 128, 8, False),
    ([130, 90], [130, 1000], 96, 1, 64, 16, True),
]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention(shape, dtype, bits):
    new, keys, Hq, Hkv, D, ps, tree = SHAPES[shape]
    d = make_batch(new, keys, Hq, Hkv, D, ps, dtype, bits, tree, seed=shape)
    out, lse = call(d)
    compare(d, out, lse)


@pytest.mark.parametrize("bits", [16, 4])
def test_tree_words_fewer_than_tokens(bits):
    """Bits past the words read as 0; a word of 0 and no context leaves the row empty."""
    d = make_batch([40, 3], [40, 50], 4, 2, 128, 16, BF, bits, True, seed=5, words=1)
    d["tree"][0] = 0
    out, lse = call(d)
    compare(d, out, lse)
    assert bool((out[0] == 0).all()) and bool(torch.isinf(lse[0]).all())


@pytest.mark.parametrize("more", [0, 60])
@pytest.mark.parametrize("bits", [16, 4])
def test_scale_strides_and_rows_of_no_sequence(bits, more):
    """Another scale; token-major pools; q and out as slices; a table with a row stride; q_starts that
    skip the first rows and end before the last."""
    from ae_b200 import paged
    d = make_batch([9 + more, 1, 4], [300, 77, 4], 8, 2, 128, 16, BF, bits, False, seed=3)
    N = 14 + more
    for name in ("k_cache", "v_cache"):
        c = d[name]
        pool = torch.zeros(c.shape[0], c.shape[2], c.shape[1] + 1, c.shape[3], dtype=c.dtype, device="cuda")
        pool[:, :, :-1] = c.transpose(1, 2)
        d[name] = pool.transpose(1, 2)[:, :-1]
    wide = torch.randn(N + 4, 8 + 3, 128, device="cuda").to(BF)
    wide[2:N + 2, 1:9] = d["q"]
    d["q"] = wide[:, 1:9]
    d["q_starts"] += 2
    table = torch.zeros(3, d["block_table"].shape[1] + 5, dtype=torch.int32, device="cuda")
    table[:, :d["block_table"].shape[1]] = d["block_table"]
    d["block_table"] = table[:, :d["block_table"].shape[1]]
    buf = torch.full((N + 4, 10, 128), 7.0, device="cuda").to(BF)
    lse = torch.full((N + 4, 8), 7.0, device="cuda")
    paged.paged_attention(d["q"], d["k_cache"], d["v_cache"], d["block_table"], d["kv_lens"], d["q_starts"],
                          scale=0.2, out=buf[:, 2:], lse=lse)
    compare(d, buf[:, 2:], lse, scale=0.2)
    assert bool((buf[:, :2] == 7.0).all())


@pytest.mark.parametrize("heads", [4, 32, 128])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("tree", [False, True])
def test_masked_places_may_hold_anything(bits, tree, heads):
    """NaN and infinities in rows past the keys, in unused pages and in new tokens that a row does not
    see leave that row's result as it was; rows that see them become NaN or infinite."""
    new, keys = [6, 3], [70, 35]
    d = make_batch(new, keys, heads, 2, 128, 16, BF, bits, tree, seed=11)
    if tree:
        sees = torch.tensor([[1, 3, 5, 9, 17, 33], [1, 3, 7, 0, 0, 0]], dtype=torch.int32, device="cuda")
        d["tree"] = torch.cat([sees[0], sees[1, :3]])[:, None].contiguous()
    good, good_lse = call(d)
    compare(d, good, good_lse)
    k, v = d["k_cache"].clone(), d["v_cache"].clone()
    kk, vv = d["k_cache"], d["v_cache"]
    D, ps = 128, 16

    def spoil(b, j, value):
        p, s = int(d["block_table"][b, j // ps]), j % ps
        for c in (kk, vv):
            if bits == 16:
                c[p, :, s] = value
            else:
                c[p, :, s, D // 2:D // 2 + D // 8] = torch.tensor([value, value] * (D // 32), dtype=BF).view(torch.uint8).cuda()

    for b in range(2):
        for j in range(keys[b], -(-keys[b] // ps) * ps):
            spoil(b, j, math.nan)
    used = torch.zeros(kk.shape[0], dtype=torch.bool, device="cuda")
    for b in range(2):
        used[d["block_table"][b, : -(-keys[b] // ps)].long()] = True
    kk[~used] = 255
    vv[~used] = 255
    out, lse = call(d)
    assert torch.equal(out, good) and torch.equal(lse, good_lse)
    # the newest token but one of sequence 0: seen by itself and what hangs below it
    spoil(0, keys[0] - 2, math.nan)
    out, lse = call(d)
    sees = [4, 5] if not tree else [4]
    for i in range(9):
        if i in sees:
            assert bool(torch.isnan(out[i]).all()), i
        else:
            assert torch.equal(out[i], good[i]) and torch.equal(lse[i], good_lse[i]), i
    # an infinite value with a finite key
    d["k_cache"].copy_(k)
    d["v_cache"].copy_(v)
    if bits == 16:
        p, s = int(d["block_table"][0, (keys[0] - 2) // ps]), (keys[0] - 2) % ps
        vv[p, :, s, 5] = math.inf
        out, _ = call(d)
        for i in range(9):
            if i in sees:
                assert bool(torch.isposinf(out[i, :, 5]).all())
                keep = [x for x in range(D) if x != 5]
                assert torch.equal(out[i][:, keep], good[i][:, keep])
            else:
                assert torch.equal(out[i], good[i]), i


@pytest.mark.parametrize("heads", [4, 48, 128])
@pytest.mark.parametrize("bits", [16, 4])
def test_bad_pages_are_left_out_and_reported(bits, heads):
    from ae_b200 import paged
    d = make_batch([2, 4], [200, 90], heads, 2, 64, 16, FP, bits, False, seed=2)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    call(d, status=status)
    assert int(status) == 0
    d["block_table"][0, 3] = d["k_cache"].shape[0]
    d["block_table"][1, 0] = -5
    out, lse = call(d, status=status)
    assert int(status) == paged.BAD_PAGE
    compare(d, out, lse)


def test_lengths_are_cut_to_the_table():
    """kv_lens past the table, q_starts past the rows."""
    d = make_batch([3, 5], [64, 48], 4, 2, 128, 16, BF, 16, False, seed=8)
    d["kv_lens"][0] = 1000
    d["block_table"][1, 3] = 0
    d["q_starts"][2] = 99
    out, lse = call(d)
    d["q_starts"][2] = 8
    compare(d, out, lse)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("new,keys", [([1] * 300, [7 + 3 * i for i in range(300)]), ([1, 1], [40000, 12]),
                                      ([600], [2000])])
def test_many_sequences_and_long_ones(new, keys, bits):
    """More sequences than the plan has threads, one long sequence over many CTAs, many row tiles."""
    d = make_batch(new, keys, 4, 1, 128, 16, BF, bits, False, seed=4)
    out, lse = call(d)
    compare(d, out, lse)
    again, lse2 = call(d)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


def test_offsets_past_32_bits():
    """A cache of 5 GB each for keys and values: rows behind 2^32 bytes."""
    from ae_b200 import paged
    Hkv, ps, D = 8, 64, 128
    pages = (5 << 30) // (Hkv * ps * D * 2)
    k = torch.empty(pages, Hkv, ps, D, dtype=BF, device="cuda")
    v = torch.empty_like(k)
    d = make_batch([1, 3], [200, 130], 16, Hkv, D, ps, BF, 16, False, seed=6)
    used = [-(-200 // ps), -(-130 // ps)]
    at = pages - 1
    table = d["block_table"].clone()
    for b in range(2):
        for i in range(used[b]):
            k[at] = d["k_cache"][int(table[b, i])]
            v[at] = d["v_cache"][int(table[b, i])]
            table[b, i] = at
            at -= 1
    small = call(d)
    d.update(k_cache=k, v_cache=v, block_table=table)
    big = call(d)
    assert torch.equal(small[0], big[0]) and torch.equal(small[1], big[1])
    x = torch.randn(1, 16 + 16, D, device="cuda").to(BF)
    slot = torch.tensor([(pages - 1) * ps + 7], device="cuda")
    paged.kv_append(x[:, :16], x[:, 16:24], x[:, 24:], k, v, slot)
    assert torch.equal(k[pages - 1, :, 7], x[0, 16:24]) and torch.equal(v[pages - 1, :, 7], x[0, 24:])



APPENDS = [
    # N, Hq, Hkv, D, ps, rot, interleaved, norm
    (1, 1, 1, 64, 1, 64, False, False),
    (3, 32, 8, 128, 16, 128, False, True),
    (77, 5, 1, 256, 32, 64, True, True),
    (50, 12, 4, 64, 64, 16, False, False),
    (129, 8, 2, 128, 8, 32, True, False),
    (5, 40, 8, 128, 16, 0, False, True),
    (600, 6, 2, 128, 128, 128, False, False),
    (9, 3, 1, 256, 16, 256, False, True),
]


def append_case(i, dtype, bits, N, Hq, Hkv, D, ps, rot, interleaved, norm):
    g = gen(100 + i)
    pages = N // ps + 3
    x = torch.randn(N, Hq + 2 * Hkv, D, generator=g, device="cuda").mul_(2).to(dtype)
    c = dict(x=x, q=x[:, :Hq], k=x[:, Hq:Hq + Hkv], v=x[:, Hq + Hkv:],
             k_cache=make_cache(g, pages, Hkv, ps, D, dtype, bits), v_cache=make_cache(g, pages, Hkv, ps, D, dtype, bits),
             slots=torch.randperm(pages * ps, generator=g, device="cuda")[:N],
             positions=torch.randint(0, 1 << 20, (N,), generator=g, device="cuda"))
    f = 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64, device="cuda") * 2 / max(rot, 1))
    c["inv_freq"] = f if rot else None
    c["w"] = [(1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(dtype) if norm else None for _ in range(2)]
    return c


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("shape", range(len(APPENDS)))
def test_append(shape, dtype, bits):
    from ae_b200 import paged
    N, Hq, Hkv, D, ps, rot, interleaved, norm = APPENDS[shape]
    c = append_case(shape, dtype, bits, *APPENDS[shape])
    drop = N > 2
    if drop:
        c["slots"][1] = -1
    before = [c["k_cache"].clone(), c["v_cache"].clone()]
    kw = dict(positions=c["positions"], inv_freq=c["inv_freq"]) if rot else {}
    out = paged.kv_append(c["q"], c["k"], c["v"], c["k_cache"], c["v_cache"], c["slots"], interleaved=interleaved,
                          rope_scale=1.25 if rot else 1.0, q_norm=c["w"][0], k_norm=c["w"][1], eps=1e-5, **kw)
    want = []
    for t, w in ((c["q"], c["w"][0]), (c["k"], c["w"][1])):
        y = t.double()
        if norm:
            y = ref.head_norm(y, w, 1e-5)
        if rot:
            y = ref.rotate(y, c["positions"], c["inv_freq"], interleaved, 1.25)
        want.append(y)
    want.append(c["v"].double())
    u = ref.half_step(dtype)

    def near(got, y, rounding):
        slack = 2.0 ** -18 * y.abs().amax(-1, keepdim=True) + 2.0 ** -25
        assert bool(((got.double() - y).abs() <= rounding + slack).all())

    near(out, want[0], u * want[0].abs())
    keep = c["slots"] >= 0
    page, at = c["slots"][keep] // ps, c["slots"][keep] % ps
    for cache, old, y in ((c["k_cache"], before[0], want[1][keep]), (c["v_cache"], before[1], want[2][keep])):
        rows = cache[page, :, at]
        if bits == 16:
            near(rows, y, u * y.abs())
        else:
            g = y.reshape(*y.shape[:-1], D // 32, 32)
            lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
            step = (hi - lo) / 15
            # half a step of the codes; scale and zero are each off by u of themselves (15 steps of the
            # scale at most), and a code at the upper end may be cut by as much
            tol = (step * (1 + u) / 2 + 15 * step * u + lo.abs() * u).expand_as(g).reshape(y.shape)
            near(ref.values(rows, D, dtype), y, tol)
            read = paged.kv4_read(cache, c["slots"], D, dtype)
            v64 = ref.values(rows, D, dtype)
            assert bool(((read[keep].double() - v64).abs() <= u * v64.abs() + 2.0 ** -24 * v64.abs().amax()).all())
            assert bool((read[~keep] == 0).all())
        untouched = torch.ones(cache.shape[0], cache.shape[2], dtype=torch.bool, device="cuda")
        untouched[page, at] = False
        sel = untouched[:, None, :, None].expand_as(cache)
        assert torch.equal(cache[sel].view(torch.uint8), old[sel].view(torch.uint8))


def test_append_codes_of_flat_and_special_groups():
    """A group of one value has scale 0 and that value as zero; codes reach both ends; non-finite
    inputs give some row, and only that row."""
    from ae_b200 import paged
    D, ps = 64, 16
    v = torch.zeros(4, 1, D, device="cuda").to(BF)
    v[0] = 3.0
    v[1, 0] = torch.arange(D, device="cuda") % 16
    v[2, 0, 3] = math.nan
    v[3, 0, 40] = math.inf
    kc, vc = (torch.zeros(2, 1, ps, ref.row_bytes(D), dtype=torch.uint8, device="cuda") for _ in range(2))
    slots = torch.tensor([5, 17, 30, 31], device="cuda")
    paged.kv_append(v.clone(), v, v, kc, vc, slots)
    got = paged.kv4_read(vc, slots, D, BF)
    assert torch.equal(got[0], v[0]) and torch.equal(got[1], v[1])
    assert torch.equal(got[2][:, 32:], v[2][:, 32:]) and torch.equal(got[3][:, :32], v[3][:, :32])
    assert int(vc[0, 0, 6:].count_nonzero()) == 0


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
def test_append_codes_are_exact(dtype):
    """Values that are not rotated are what they are: the rows are those of the 64-bit form byte for byte,
    ties between two codes (half even) among them.  (A scale may be off by a last place where its 32-bit
    quotient falls on the middle of two 16-bit numbers, 2^-12 of them at most; such groups are left out.)"""
    from ae_b200 import paged
    D, N = 128, 2000
    v = torch.randn(N, 4, D, generator=gen(5), device="cuda").to(dtype)
    v[::3] = (v[::3] * 8).round() / 8  # many ties
    kc, vc = (torch.zeros(N // 16 + 1, 4, 16, ref.row_bytes(D), dtype=torch.uint8, device="cuda") for _ in range(2))
    slots = torch.arange(N, device="cuda")
    paged.kv_append(v.clone(), v, v, kc, vc, slots)
    want, _ = ref.quantise(v.double(), dtype)
    for c in (kc, vc):
        got = c[slots // 16, :, slots % 16]
        sz = lambda x: x[..., D // 2:D // 2 + D // 8].reshape(N, 4, D // 32, 4)  # noqa: E731
        codes = lambda x: x[..., :D // 2].reshape(N, 4, D // 32, 16)  # noqa: E731
        same = (sz(got) == sz(want)).all(-1)
        assert float(same.double().mean()) >= 1 - 2 ** -12
        assert torch.equal(codes(got)[same], codes(want)[same])


def test_append_slots_outside():
    from ae_b200 import paged
    c = append_case(0, BF, 16, 6, 4, 2, 64, 16, 64, False, False)
    c["slots"][:] = torch.tensor([0, -1, 10 ** 12, c["k_cache"].shape[0] * 16, 7, -9], device="cuda")
    old = c["k_cache"].clone()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    paged.kv_append(c["q"], c["k"], c["v"], c["k_cache"], c["v_cache"], c["slots"], status=status)
    assert int(status) == paged.BAD_PAGE
    old[0, :, 0], old[0, :, 7] = c["k"][0], c["k"][4]
    assert torch.equal(old, c["k_cache"])
    got = paged.kv4_read(torch.full((2, 1, 16, 48), 255, dtype=torch.uint8, device="cuda"),
                         torch.tensor([-1, 32, 10 ** 14], device="cuda"), 64, BF)
    assert bool((got == 0).all())


@pytest.mark.parametrize("bits", [16, 4])
def test_append_then_attend_captured_and_on_another_stream(bits):
    """The two as a decode step uses them: eagerly, captured in two graphs whose replays overlap, and on
    another stream, with the same results."""
    from ae_b200 import paged
    B, Hq, Hkv, D, ps = 3, 8, 2, 128, 16
    states = []
    for seed in (0, 1):
        d = make_batch([4] * B, [40, 500, 2100], Hq, Hkv, D, ps, BF, bits, True, seed=seed)
        g = gen(50 + seed)
        x = torch.randn(4 * B, Hq + 2 * Hkv, D, generator=g, device="cuda").to(BF)
        lens = d["kv_lens"].tolist()
        pos = torch.tensor([lens[b] - 4 + i for b in range(B) for i in range(4)], device="cuda")
        slots = torch.stack([d["block_table"][i // 4, int(p) // ps].long() * ps + int(p) % ps for i, p in enumerate(pos)])
        f, s = paged.rope_inv_freq(D, 1e6, "yarn", 4.0, device="cuda")
        states.append((d, x, pos, slots, f, s))

    def step(st):
        d, x, pos, slots, f, s = st
        q = paged.kv_append(x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], d["k_cache"], d["v_cache"], slots, pos, f, rope_scale=s)
        return q, paged.paged_attention(q, d["k_cache"], d["v_cache"], d["block_table"], d["kv_lens"], d["q_starts"], tree=d["tree"])

    want = [step(st)[1].clone() for st in states]
    for st, w in zip(states, want):
        d = dict(st[0])
        d["q"] = step(st)[0]
        lse = torch.empty(d["q"].shape[:2], device="cuda")
        out = paged.paged_attention(d["q"], d["k_cache"], d["v_cache"], d["block_table"], d["kv_lens"], d["q_starts"],
                                    tree=d["tree"], lse=lse)
        compare(d, out, lse)
        assert torch.equal(out, w)
    graphs = []
    for st in states:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = step(st)[1]
        graphs.append((gr, res))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for (gr, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    for (_, res), w in zip(graphs, want):
        assert torch.equal(res, w)
    with torch.cuda.stream(streams[0]):
        other = step(states[0])[1]
    streams[0].synchronize()
    assert torch.equal(other, want[0])


def test_no_tokens_and_no_sequences():
    from ae_b200 import paged
    d = make_batch([1], [5], 4, 2, 64, 16, BF, 16, False)
    e = torch.zeros(0, 4, 64, dtype=BF, device="cuda")
    z = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = paged.paged_attention(e, d["k_cache"], d["v_cache"], d["block_table"][:0], z[:0], z)
    assert out.shape == (0, 4, 64)
    lse = torch.full((1, 4), 7.0, device="cuda")
    keep = torch.full((1, 4, 64), 7.0, device="cuda").to(BF)
    paged.paged_attention(d["q"], d["k_cache"], d["v_cache"], d["block_table"][:0], z[:0], z, out=keep, lse=lse)
    assert bool((keep == 7).all()) and bool((lse == 7).all())
    kv = torch.zeros(0, 2, 64, dtype=BF, device="cuda")
    q = paged.kv_append(e, kv, kv, d["k_cache"], d["v_cache"], torch.zeros(0, dtype=torch.int64, device="cuda"))
    assert q.shape == (0, 4, 64)


def test_same_bits_again_and_again():
    """Every kernel path, repeated among other work: the same bits each time."""
    picks = [0, 3, 5, 6, 10, 11, 13, 14, 15, 16, 17, 18, 20]
    cases = []
    for bits in (16, 4):
        for i in picks:
            new, keys, Hq, Hkv, D, ps, tree = SHAPES[i]
            cases.append(make_batch(new, keys, Hq, Hkv, D, ps, BF if i % 2 else FP, bits, tree, seed=i))
    first = [call(d) for d in cases]
    junk = torch.empty(16 << 20, device="cuda")
    for r in range(25):
        for n, d in enumerate(cases):
            out, lse = call(d)
            assert torch.equal(out, first[n][0]) and torch.equal(lse, first[n][1]), (n, r)
            if n % 5 == r % 5:
                junk.fill_(math.nan)


def test_two_streams_at_once():
    """Calls on two streams overlap without a shared workspace."""
    cases = [make_batch([32] * 4, [900, 33, 2000, 64], 8, 2, 128, 16, BF, bits, True, seed=bits) for bits in (16, 4)]
    want = [call(d) for d in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (d, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i].append(call(d))
    torch.cuda.synchronize()
    for i in range(2):
        for out, lse in got[i]:
            assert torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])


def test_long_rows_of_scores_far_apart():
    """Scores that grow along the keys by hundreds: every tile raises the maximum."""
    for bits, heads in ((16, 4), (16, 64), (4, 4)):
        d = make_batch([2], [700], heads, 2, 128, 16, BF, bits, False, seed=1)
        if bits == 16:
            ramp = torch.linspace(-3, 3, d["k_cache"].shape[0] * 16, device="cuda").view(-1, 1, 16, 1)
            d["k_cache"] = (d["k_cache"] * 0.1 + d["q"][0, 0] * ramp).to(BF)
        d["q"] = (d["q"] * 6).to(BF)
        out, lse = call(d)
        o, l, spread, _ = ref.attention(d["q"], d["k_cache"], d["v_cache"], d["block_table"], d["kv_lens"], d["q_starts"])
        # scores of up to a thousand: 32 bits hold them to 2^-14
        u = ref.half_step(BF)
        assert bool(((out.double() - o).abs() <= 2 * u * spread + u * o.abs() + 2 ** -11 * spread + 2 ** -25).all())
        assert bool(((lse.double() - l).abs() <= 2 ** -17 * l.abs() + 2 ** -13).all())


@pytest.mark.parametrize("change", [
    dict(q=lambda d: d["q"].float()), dict(q=lambda d: d["q"][:, 0]), dict(q=lambda d: d["q"][..., :64]),
    dict(q=lambda d: d["q"].transpose(1, 2).contiguous().transpose(1, 2)), dict(q=lambda d: d["q"][:, :3]),
    dict(k_cache=lambda d: d["k_cache"][:, :, :12]), dict(k_cache=lambda d: d["k_cache"].half()),
    dict(k_cache=lambda d: d["k_cache"].transpose(1, 2).contiguous().transpose(1, 2)),
    dict(block_table=lambda d: d["block_table"].long()), dict(block_table=lambda d: d["block_table"].cpu()),
    dict(kv_lens=lambda d: d["kv_lens"].long()), dict(kv_lens=lambda d: d["kv_lens"][:1]),
    dict(q_starts=lambda d: d["q_starts"][:2]), dict(q_starts=lambda d: d["q_starts"].cpu()),
    dict(tree=lambda d: torch.zeros(3, 1, dtype=torch.int32, device="cuda")),
    dict(tree=lambda d: torch.zeros(4, 0, dtype=torch.int32, device="cuda")),
    dict(tree=lambda d: torch.zeros(4, 1, dtype=torch.int64, device="cuda"))])
def test_attention_refusals(change):
    from ae_b200 import paged
    d = make_batch([3, 1], [40, 7], 4, 2, 128, 16, BF, 16, False)
    for name, f in change.items():
        d[name] = f(d)
    with pytest.raises((ValueError, NotImplementedError)):
        paged.paged_attention(**d)


@pytest.mark.parametrize("kw", [dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan),
                                dict(lse=torch.zeros(4, 4)), dict(out=torch.zeros(4, 4, 128)),
                                dict(status=torch.zeros(1))])
def test_attention_option_refusals(kw):
    from ae_b200 import paged
    d = make_batch([3, 1], [40, 7], 4, 2, 128, 16, BF, 16, False)
    with pytest.raises(ValueError):
        paged.paged_attention(**d, **kw)
    with pytest.raises(ValueError):
        paged.paged_attention(**d, out=d["q"])
    d["k_cache"], d["v_cache"] = d["k_cache"][:0], d["v_cache"][:0]
    with pytest.raises(ValueError):
        paged.paged_attention(**d)


@pytest.mark.parametrize("strides,good", [((512, 128), True), ((128, 512), True), ((640, 136), True), ((0, 128), False),
                                          ((128, 128), False), ((512, 0), False), ((256, 128), False), ((512, 64), False)])
def test_rows_of_out_may_not_overlap(strides, good):
    from ae_b200 import paged
    d = make_batch([3, 1], [40, 7], 4, 2, 128, 16, BF, 16, False)
    out = torch.zeros(4096, dtype=BF, device="cuda").as_strided((4, 4, 128), (*strides, 1))
    if good:
        assert torch.equal(paged.paged_attention(**d, out=out), paged.paged_attention(**d))
    else:
        with pytest.raises(ValueError, match="overlap"):
            paged.paged_attention(**d, out=out)


def test_tables_of_more_than_30_bits_are_refused():
    from ae_b200 import paged
    d = make_batch([1], [40], 4, 2, 64, 16, BF, 16, False)
    d["k_cache"], d["v_cache"] = paged.new_cache(1, 2, 65536, 64, BF, "cuda")
    d["block_table"] = torch.zeros(1, (1 << 14) + 1, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="2\\^30"):
        paged.paged_attention(**d)
    d["block_table"] = d["block_table"][:, :-1]
    assert torch.isfinite(paged.paged_attention(**d)).all()


@pytest.mark.parametrize("change", [
    dict(k=lambda c: c["k"][:, :1]), dict(v=lambda c: c["v"].float()), dict(slots=lambda c: c["slots"].int()),
    dict(slots=lambda c: c["slots"][:-1]), dict(positions=lambda c: c["positions"].int()),
    dict(inv_freq=lambda c: c["inv_freq"].float()), dict(inv_freq=lambda c: c["inv_freq"][:5]),
    dict(inv_freq=lambda c: None), dict(inv_freq=lambda c: torch.ones(64, dtype=torch.float64, device="cuda")),
    dict(q=lambda c: c["x"][:, :4, 1:]), dict(q=lambda c: c["q"].cpu()), dict(k_cache=lambda c: c["k_cache"][:1]),
    dict(out=lambda c: torch.zeros(6, 4, 64, device="cuda")), dict(q_norm=lambda c: torch.ones(32, device="cuda"))])
def test_append_refusals(change):
    from ae_b200 import paged
    c = append_case(0, BF, 16, 6, 4, 2, 64, 16, 64, False, False)
    for name, f in change.items():
        c[name] = f(c)
    c.pop("x"), c.pop("w")
    with pytest.raises((ValueError, NotImplementedError)):
        paged.kv_append(**c)
