"""Cases of the paged key/value cache and the attention over it, with their plain forms.

Three operators of ``ae_b200.paged``: ``kv_append`` (norm of each head, rotary positions and the
write into a paged cache, of 16-bit values or of 4-bit codes), and ``paged_attention`` over a
16-bit cache and over a 4-bit one.  ``run`` computes the plain form with elementary torch
operations where ``own`` is false and calls the framework where it is true."""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # the tokens of one decode step of four sequences: latency
        dict(name="append decode", op="append", bits=16, N=4, Hq=32, Hkv=8, D=128, ps=16, dtype="bf16", rot=128,
             interleaved=False, scaling="none", norm=False),
        # a prefill chunk, an odd number of tokens, with the norm of each head
        dict(name="append prefill", op="append", bits=16, N=8199, Hq=32, Hkv=8, D=128, ps=64, dtype="bf16", rot=128,
             interleaved=False, scaling="none", norm=True),
        # wide heads of which a quarter is rotated, in adjacent pairs, positions stretched
        dict(name="append partial", op="append", bits=16, N=1023, Hq=16, Hkv=4, D=256, ps=32, dtype="fp16", rot=64,
             interleaved=True, scaling="linear", norm=False),
        # a prefill chunk into a 4-bit cache, and the rows read back
        dict(name="append 4-bit", op="append", bits=4, N=4095, Hq=48, Hkv=8, D=128, ps=64, dtype="bf16", rot=128,
             interleaved=False, scaling="yarn", norm=True),
        # one token for each of four short sequences: latency
        dict(name="decode short", op="attend", bits=16, B=4, n=1, kv=640, ragged=True, mode="causal", Hq=32, Hkv=8,
             D=128, ps=16, dtype="bf16"),
        # the verify step of the benchmark: four sequences, trees of 32 draft tokens, 2048 tokens of context
        dict(name="verify", op="attend", bits=16, B=4, n=32, kv=2080, ragged=False, mode="tree", Hq=32, Hkv=8, D=128,
             ps=64, dtype="bf16"),
        # verify over long, ragged contexts, with six query heads to a key head
        dict(name="verify long", op="attend", bits=16, B=16, n=32, kv=16384, ragged=True, mode="tree", Hq=48, Hkv=8,
             D=128, ps=32, dtype="bf16"),
        # one token for each of 32 long sequences: memory
        dict(name="decode long", op="attend", bits=16, B=32, n=1, kv=32768, ragged=True, mode="causal", Hq=32, Hkv=8,
             D=128, ps=16, dtype="fp16"),
        # chunks of two long prompts: arithmetic
        dict(name="prefill chunk", op="attend", bits=16, B=2, n=2048, kv=8191, ragged=True, mode="causal", Hq=32,
             Hkv=8, D=128, ps=128, dtype="bf16"),
        # one token for each of eight sequences over a 4-bit cache with narrow heads: latency
        dict(name="decode short 4-bit", op="attend", bits=4, B=8, n=1, kv=1001, ragged=True, mode="causal", Hq=32,
             Hkv=8, D=64, ps=16, dtype="fp16"),
        # verify over long contexts in a 4-bit cache
        dict(name="verify long 4-bit", op="attend", bits=4, B=16, n=32, kv=16384, ragged=True, mode="tree", Hq=32,
             Hkv=8, D=128, ps=64, dtype="bf16"),
        # one token for each of 32 long sequences over a 4-bit cache: memory
        dict(name="decode long 4-bit", op="attend", bits=4, B=32, n=1, kv=32768, ragged=True, mode="causal", Hq=32,
             Hkv=8, D=128, ps=32, dtype="bf16"),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    bits = rng.choice((16, 4))
    D = rng.choice((64, 128, 128, 256))
    Hkv = rng.choice((1, 2, 4, 8))
    c = dict(bits=bits, Hq=Hkv * rng.choice((1, 2, 4, 5, 6, 8)), Hkv=Hkv, D=D, ps=rng.choice((1, 8, 16, 32, 64, 128)),
             dtype=rng.choice(("bf16", "fp16")))
    if rng.random() < 0.35:
        return dict(c, op="append", N=_log_uniform(rng, 1, 8000), rot=rng.choice((16, D // 4, D // 2, D)),
                    interleaved=rng.random() < 0.5, scaling=rng.choice(("none", "linear", "yarn")),
                    norm=rng.random() < 0.5)
    kind = rng.choice(("decode", "verify", "prefill"))
    if kind == "prefill":
        B, n = rng.randint(1, 3), _log_uniform(rng, 65, 1500)
    elif kind == "verify":
        B, n = _log_uniform(rng, 1, 24), rng.randint(2, 64)
    else:
        B, n = _log_uniform(rng, 1, 48), 1
    most = {"decode": 32768, "verify": 12000, "prefill": 6000}[kind]
    kv = _log_uniform(rng, n, most)
    c = dict(c, op="attend", B=B, n=n, kv=kv, ragged=rng.random() < 0.7, mode="tree" if kind == "verify" else "causal")
    while c["B"] * c["kv"] * Hkv * D > 300_000_000 or work(c)["flops"] > 2.5e11:  # the largest listed case is larger
        if c["B"] > 1:
            c["B"] -= 1
        else:
            c["n"], c["kv"] = c["n"] // 2 + 1, c["kv"] // 2 + 1
    return c


def _lengths(case):
    """Per sequence: new tokens and keys (the new ones among them), the same for every seed."""
    rng = random.Random(case["B"] * 1000003 + case["kv"])
    new, keys = [], []
    for b in range(case["B"]):
        n, kv = case["n"], case["kv"]
        if case["ragged"] and b > 0:
            n = rng.randint(max(1, n // 2), n)
            kv = rng.randint(max(n, kv // 4), kv)
        new.append(n)
        keys.append(kv)
    return new, keys


def _row_bytes(D):
    return (D // 2 + D // 8 + 15) // 16 * 16


def _inv_freq(case):
    """Angle of each rotated pair at position 1, in 64 bits, and the factor on cos and sin."""
    r, base, factor, trained = case["rot"], 1e6, 4.0, 8192
    f = torch.tensor([base ** (-2.0 * i / r) for i in range(r // 2)], dtype=torch.float64)
    if case["scaling"] == "linear":
        return f / factor, 1.0
    if case["scaling"] == "yarn":
        # frequencies that turn often within the trained length stay, slow ones are stretched
        turns = trained * f / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        return f * keep + f / factor * (1 - keep), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _quantise(x, dtype):
    """Rows [..., D] of a 4-bit cache from values of 32 bits."""
    D = x.shape[-1]
    g = x.reshape(*x.shape[:-1], D // 32, 32)
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale, zero = ((hi - lo) / 15.0).to(dtype), lo.to(dtype)
    s, z = scale.to(x.dtype), zero.to(x.dtype)
    code = torch.where(s > 0, ((g - z) / s).round().clamp(0, 15), torch.zeros_like(g)).to(torch.uint8)
    code = code.reshape(*x.shape[:-1], D // 2, 2)
    rows = torch.zeros(*x.shape[:-1], _row_bytes(D), dtype=torch.uint8, device=x.device)
    rows[..., : D // 2] = code[..., 0] | (code[..., 1] << 4)
    rows[..., D // 2: D // 2 + D // 8] = torch.cat([scale, zero], -1).flatten(-2).contiguous().view(torch.uint8)
    return rows


def _values(rows, D, dtype):
    """The 32-bit values that rows of a 4-bit cache stand for."""
    codes = rows[..., : D // 2]
    codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    sz = rows[..., D // 2: D // 2 + D // 8].contiguous().view(dtype).float()
    sz = sz.reshape(*rows.shape[:-1], D // 32, 2)
    codes = codes.reshape(*rows.shape[:-1], D // 32, 32)
    return (codes * sz[..., :1] + sz[..., 1:]).flatten(-2)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, D, Hq, Hkv, ps = DTYPES[case["dtype"]], case["D"], case["Hq"], case["Hkv"], case["ps"]

    def rnd(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def cache(pages):
        if case["bits"] == 16:
            return torch.randn(pages, Hkv, ps, D, generator=g, device="cuda", dtype=dtype)
        rows = torch.empty(pages, Hkv, ps, _row_bytes(D), dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 26) // (Hkv * ps * D))
        for p in range(0, pages, step):
            q = min(pages, p + step)
            rows[p:q] = _quantise(rnd(q - p, Hkv, ps, D), dtype)
        return rows

    s = {"case": case, "dtype": dtype}
    if case["op"] == "append":
        N = case["N"]
        pages = -(-N // ps) + 3
        s["qkv"] = (rnd(N, (Hq + 2 * Hkv) * D) * 2).to(dtype)  # as the projection leaves it
        s["k_cache"], s["v_cache"] = cache(pages), cache(pages)
        s["slots"] = torch.randperm(pages * ps, generator=g, device="cuda")[:N]
        s["positions"] = torch.randint(0, 131072, (N,), generator=g, device="cuda")
        f, s["rope_scale"] = _inv_freq(case)
        s["inv_freq"] = f.cuda()
        s["q_norm"] = (1 + 0.1 * rnd(D)).to(dtype) if case["norm"] else None
        s["k_norm"] = (1 + 0.1 * rnd(D)).to(dtype) if case["norm"] else None
        return s
    new, keys = _lengths(case)
    width = -(-max(keys) // ps)
    used = [-(-k // ps) for k in keys]
    pages = sum(used) + 2
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(case["B"], width, dtype=torch.int32, device="cuda")
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = order[at:at + u]
        at += u
    N = sum(new)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s["q"] = (rnd(N, Hq, D) * 1.5).to(dtype)
    s["k_cache"], s["v_cache"] = cache(pages), cache(pages)
    s["table"] = table
    s["kv_lens"] = torch.tensor(keys, dtype=torch.int32, device="cuda")
    s["q_starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s["most_new"], s["tree"] = max(new), None
    if case["mode"] == "tree":
        # a random draft tree for each sequence: token i hangs below an earlier one or below the context
        words = -(-max(new) // 32)
        rng = random.Random(seed)
        masks = []
        for n in new:
            sees = []
            for i in range(n):
                p = rng.randint(-1, i - 1)
                sees.append((sees[p] if p >= 0 else 0) | 1 << i)
            for m in sees:
                row = [(m >> (32 * w)) & 0xFFFFFFFF for w in range(words)]
                masks.append([v - (1 << 32) if v >> 31 else v for v in row])
        s["tree"] = torch.tensor(masks, dtype=torch.int32, device="cuda")
    return s


def _plain_append(s):
    c, dtype = s["case"], s["dtype"]
    N, Hq, Hkv, D, r = c["N"], c["Hq"], c["Hkv"], c["D"], c["rot"]
    x = s["qkv"].float().view(N, Hq + 2 * Hkv, D)
    q, k, v = x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]
    if c["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-6) * s["q_norm"].float()
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + 1e-6) * s["k_norm"].float()
    angle = s["positions"].double()[:, None, None] * s["inv_freq"]
    cos, sin = (angle.cos() * s["rope_scale"]).float(), (angle.sin() * s["rope_scale"]).float()

    def rotate(t):
        if c["interleaved"]:
            a, b = t[..., 0:r:2], t[..., 1:r:2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = t[..., : r // 2], t[..., r // 2:r]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([turned, t[..., r:]], -1)

    q, k = rotate(q), rotate(k)
    page, at = s["slots"] // c["ps"], s["slots"] % c["ps"]
    if c["bits"] == 16:
        s["k_cache"][page, :, at] = k.to(dtype)
        s["v_cache"][page, :, at] = v.to(dtype)
        return q.to(dtype), s["k_cache"], s["v_cache"]
    s["k_cache"][page, :, at] = _quantise(k, dtype)
    s["v_cache"][page, :, at] = _quantise(v, dtype)
    return (q.to(dtype), _values(s["k_cache"][page, :, at], D, dtype).to(dtype),
            _values(s["v_cache"][page, :, at], D, dtype).to(dtype))


def _plain_attend(s):
    c, dtype = s["case"], s["dtype"]
    B, Hq, Hkv, D, n = c["B"], c["Hq"], c["Hkv"], c["D"], s["most_new"]
    table = s["table"].long()
    S = table.shape[1] * c["ps"]

    def keys_of(cache):  # [B, Hkv, S, D] in 32 bits
        x = cache[table].transpose(1, 2).reshape(B, Hkv, S, -1)
        return x.float() if c["bits"] == 16 else _values(x, D, dtype)

    starts, lens = s["q_starts"].long(), s["kv_lens"].long()
    count = starts[1:] - starts[:-1]
    i = torch.arange(n, device="cuda")
    there = i < count[:, None]                                    # [B, n]
    row = (starts[:-1, None] + i).clamp_(max=s["q"].shape[0] - 1)
    q = s["q"][row].float().view(B, n, Hkv, Hq // Hkv, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, D)
    score = (q @ keys_of(s["k_cache"]).transpose(-1, -2)) * D ** -0.5
    j = torch.arange(S, device="cuda")
    local = j - (lens - count)[:, None]                           # [B, S]: place among the new tokens
    if s["tree"] is None:
        sees = local[:, None, :] <= i[:, None]
    else:
        bits = s["tree"][row].long()                              # [B, n, words]
        word = (local.clamp(min=0) // 32).clamp(max=bits.shape[-1] - 1)
        bit = bits.gather(-1, word[:, None, :].expand(B, n, S)) >> (local.clamp(min=0) % 32)[:, None, :]
        sees = (local[:, None, :] < 0) | ((bit & 1) != 0)
    sees = (sees & (j < lens[:, None])[:, None, :])[:, None, :, None, :].expand(B, 1, n, Hq // Hkv, S)
    score = score.masked_fill_(~sees.reshape(B, 1, -1, S), -math.inf)
    top = score.amax(-1, keepdim=True)
    p = (score - top.clamp(min=-3e38)).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p @ keys_of(s["v_cache"])) / total.clamp(min=1e-30)
    o = o.view(B, Hkv, n, Hq // Hkv, D).permute(0, 2, 1, 3, 4).reshape(B, n, Hq, D)[there].to(dtype)
    if c["bits"] == 4:
        return o
    lse = (top + total.log()).view(B, Hkv, n, Hq // Hkv).transpose(1, 2).reshape(B, n, Hq)[there]
    return o, lse


def run(state):
    c = state["case"]
    if not own:
        return _plain_append(state) if c["op"] == "append" else _plain_attend(state)
    from ae_b200 import paged

    if c["op"] == "append":
        N, Hq, Hkv, D = c["N"], c["Hq"], c["Hkv"], c["D"]
        x = state["qkv"].view(N, Hq + 2 * Hkv, D)
        q = paged.kv_append(x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], state["k_cache"], state["v_cache"],
                            state["slots"], positions=state["positions"], inv_freq=state["inv_freq"],
                            interleaved=c["interleaved"], rope_scale=state["rope_scale"], q_norm=state["q_norm"],
                            k_norm=state["k_norm"], eps=1e-6)
        if c["bits"] == 16:
            return q, state["k_cache"], state["v_cache"]
        return (q, paged.kv4_read(state["k_cache"], state["slots"], D, state["dtype"]),
                paged.kv4_read(state["v_cache"], state["slots"], D, state["dtype"]))
    if c["bits"] == 4:
        return paged.paged_attention(state["q"], state["k_cache"], state["v_cache"], state["table"], state["kv_lens"],
                                     state["q_starts"], tree=state["tree"])
    lse = torch.empty(state["q"].shape[:2], dtype=torch.float32, device=state["q"].device)
    out = paged.paged_attention(state["q"], state["k_cache"], state["v_cache"], state["table"], state["kv_lens"],
                                state["q_starts"], tree=state["tree"], lse=lse)
    return out, lse


def work(case):
    D, Hq, Hkv = case["D"], case["Hq"], case["Hkv"]
    row = 2 * D if case["bits"] == 16 else D // 2 + D // 8
    if case["op"] == "append":
        N = case["N"]
        there = N * ((Hq + 2 * Hkv) * D * 2 + 16)
        back = N * (Hq * D * 2 + 2 * Hkv * row)
        if case["bits"] == 4:
            back += N * 2 * Hkv * (row + 2 * D)
        flops = N * (Hq + Hkv) * (3 * case["rot"] + (4 * D if case["norm"] else 0))
        return {"bytes": there + back, "flops": flops}
    new, keys = _lengths(case)
    seen = 0
    for n, kv in zip(new, keys):
        # a tree's token sees the context and, of the new tokens, its few ancestors at least
        seen += n * (kv - n) + (n if case["mode"] == "tree" else n * (n + 1) // 2)
    N = sum(new)
    read = sum(keys) * Hkv * 2 * row + N * Hq * D * 2 + 4 * sum(-(-k // case["ps"]) for k in keys)
    return {"bytes": read + N * Hq * (D * 2 + (4 if case["bits"] == 16 else 0)), "flops": 4 * D * Hq * seen}


def _exact_row_values(rows, D, dtype):
    out = torch.empty(*rows.shape[:-1], D, dtype=torch.float64, device=rows.device)
    sz = rows[..., D // 2: D // 2 + D // 8].contiguous().view(dtype).double()
    for d in range(D):
        code = (rows[..., d // 2] >> (4 * (d % 2))) % 16
        out[..., d] = sz[..., 2 * (d // 32)] * code.double() + sz[..., 2 * (d // 32) + 1]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    dtype, D, Hq, Hkv, ps = s["dtype"], case["D"], case["Hq"], case["Hkv"], case["ps"]
    if case["op"] == "append":
        N, r = case["N"], case["rot"]
        x = s["qkv"].double().reshape(N, Hq + 2 * Hkv, D)
        for lo, hi, w in ((0, Hq, s["q_norm"]), (Hq, Hq + Hkv, s["k_norm"])):
            if w is not None:
                part = x[:, lo:hi]
                x[:, lo:hi] = part / ((part * part).sum(-1, keepdim=True) / D + 1e-6).sqrt() * w.double()
        turn = torch.polar(torch.full((N, r // 2), float(s["rope_scale"]), dtype=torch.float64, device="cuda"),
                           s["positions"].double()[:, None] * s["inv_freq"][None, :])
        i = torch.arange(r // 2, device="cuda")
        first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + r // 2)
        z = torch.complex(x[:, :Hq + Hkv, first], x[:, :Hq + Hkv, second]) * turn[:, None, :]
        x[:, :Hq + Hkv, first], x[:, :Hq + Hkv, second] = z.real, z.imag
        q, k, v = x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]
        if case["bits"] == 4:
            outs = [q]
            for t in (k, v):
                g = t.reshape(N, Hkv, D // 32, 32)
                low = g.min(-1, keepdim=True).values
                scale = ((g.max(-1, keepdim=True).values - low) / 15).to(dtype).double()
                zero = low.to(dtype).double()
                code = torch.clamp(torch.round((g - zero) / torch.where(scale > 0, scale, 1.0)), 0, 15)
                outs.append((torch.where(scale > 0, code, 0.0) * scale + zero).reshape(N, Hkv, D))
            return tuple(outs)
        outs = [q]
        for t, cache in ((k, s["k_cache"]), (v, s["v_cache"])):
            flat = cache.double().transpose(1, 2).reshape(-1, Hkv, D)
            flat[s["slots"]] = t
            outs.append(flat.view(-1, ps, Hkv, D).transpose(1, 2))
        return tuple(outs)
    new, keys = _lengths(case)
    outs, logs, at = [], [], 0
    for b, (n, kv) in enumerate(zip(new, keys)):
        page = s["table"][b, : -(-kv // ps)].long()

        def rows_of(cache):
            x = cache[page].transpose(0, 1).reshape(Hkv, -1, cache.shape[-1])[:, :kv]
            return x.double() if case["bits"] == 16 else _exact_row_values(x, D, dtype)

        K, V = rows_of(s["k_cache"]), rows_of(s["v_cache"])
        allowed = torch.ones(n, kv, dtype=torch.bool, device="cuda")
        if s["tree"] is None:
            allowed[:, kv - n:] = torch.tril(allowed[:, kv - n:])
        else:
            for t in range(n):
                allowed[:, kv - n + t] = (s["tree"][at:at + n, t // 32].long() >> (t % 32)) % 2 == 1
        out = torch.empty(n, Hq, D, dtype=torch.float64, device="cuda")
        lse = torch.empty(n, Hq, dtype=torch.float64, device="cuda")
        for h in range(Hq):
            w = s["q"][at:at + n, h].double() @ K[h * Hkv // Hq].T / math.sqrt(D)
            w[~allowed] = -math.inf
            lse[:, h] = torch.logsumexp(w, 1)
            out[:, h] = torch.softmax(w, 1) @ V[h * Hkv // Hq]
        outs.append(out)
        logs.append(lse)
        at += n
    return torch.cat(outs) if case["bits"] == 4 else (torch.cat(outs), torch.cat(logs))
