"""Plain 64-bit forms of the paged cache operators (ae_b200/paged.py), written from their
definitions: loops over sequences, no shared code with the library."""
import math

import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def row_bytes(D):
    return -(-(D // 2 + D // 8) // 16) * 16


def quantise(x, dtype):
    """4-bit rows [..., row_bytes(D)] of values [..., D] (64 bits), and the values they stand for."""
    D = x.shape[-1]
    g = x.reshape(*x.shape[:-1], D // 32, 32)
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s, z = ((hi - lo) / 15).to(dtype), lo.to(dtype)
    code = ((g - z.double()) / torch.where(s > 0, s, torch.ones_like(s)).double()).round().clamp(0, 15)
    code = torch.where(s > 0, code, torch.zeros_like(code))
    vals = (code * s.double() + z.double()).reshape(x.shape)
    c = code.to(torch.uint8).reshape(*x.shape[:-1], D // 2, 2)
    rows = torch.zeros(*x.shape[:-1], row_bytes(D), dtype=torch.uint8, device=x.device)
    rows[..., :D // 2] = c[..., 0] + 16 * c[..., 1]
    sz = torch.cat([s, z], -1).reshape(*x.shape[:-1], D // 16).contiguous()
    rows[..., D // 2:D // 2 + D // 8] = sz.view(torch.uint8)
    return rows, vals


def values(rows, D, dtype):
    """The 64-bit values of 4-bit rows."""
    c = rows[..., :D // 2].to(torch.int64)
    c = torch.stack([c % 16, c // 16], -1).reshape(*rows.shape[:-1], D // 32, 32).double()
    sz = rows[..., D // 2:D // 2 + D // 8].contiguous().view(dtype).double().reshape(*rows.shape[:-1], D // 32, 2)
    return (c * sz[..., :1] + sz[..., 1:]).reshape(*rows.shape[:-1], D)


def rotate(x, positions, inv_freq, interleaved, scale):
    """x [N, heads, D] in 64 bits."""
    r = 2 * inv_freq.numel()
    ang = positions.double()[:, None] * inv_freq.double()[None, :]
    c, s = ang.cos()[:, None, :] * scale, ang.sin()[:, None, :] * scale
    y = x.clone()
    i = torch.arange(r // 2, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def head_norm(x, w, eps):
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()


def attention(q, k_cache, v_cache, table, kv_lens, q_starts, tree=None, scale=None, pages_ok=None):
    """(out, lse, spread, reach): out [N, Hq, D] and lse [N, Hq] in 64 bits, NaN in rows of no sequence;
    spread [N, Hq, D] = sum_j p_j |v_j|, what roundings of p and v are relative to; reach [N, Hq] =
    max_j scale sum_d |q_d k_jd|, what roundings of k are relative to."""
    dtype = q.dtype
    N, Hq, D = q.shape
    P, Hkv, ps, _ = k_cache.shape
    scale = D ** -0.5 if scale is None else scale
    out = torch.full((N, Hq, D), math.nan, dtype=torch.float64, device=q.device)
    spread = out.clone()
    lse = torch.full((N, Hq), math.nan, dtype=torch.float64, device=q.device)
    reach = torch.zeros((N, Hq), dtype=torch.float64, device=q.device)
    starts, lens = q_starts.tolist(), kv_lens.tolist()
    for b in range(len(lens)):
        s0, s1 = starts[b], min(starts[b + 1], N)
        n, L = s1 - s0, min(lens[b], table.shape[1] * ps)
        if n <= 0:
            continue
        pages = table[b, : -(-L // ps)].long()
        ok = ((pages >= 0) & (pages < P)).repeat_interleave(ps)[:L]
        pages = pages.clamp(0, P - 1)

        def rows(cache):
            x = cache[pages].transpose(1, 2).reshape(-1, Hkv, cache.shape[-1])[:L]
            return values(x, D, dtype) if cache.dtype == torch.uint8 else x.double()

        K, V = rows(k_cache), rows(v_cache)
        j = torch.arange(L, device=q.device)
        for i in range(n):
            t = j - (L - n)
            if tree is None:
                see = t <= i
            else:
                w = tree[s0 + i].tolist()
                see = torch.tensor([x < 0 or (x // 32 < len(w) and (w[x // 32] >> (x % 32)) & 1 == 1)
                                    for x in t.tolist()], dtype=torch.bool, device=q.device)
            see = see & ok
            Ks, Vs = K[see], V[see]
            for h in range(Hkv):
                hs = slice(h * (Hq // Hkv), (h + 1) * (Hq // Hkv))
                if Ks.shape[0] == 0:
                    out[s0 + i, hs], spread[s0 + i, hs], lse[s0 + i, hs] = 0, 0, -math.inf
                    continue
                sc = q[s0 + i, hs].double() @ Ks[:, h].T * scale
                p = torch.softmax(sc, -1)
                reach[s0 + i, hs] = (q[s0 + i, hs].double().abs() @ Ks[:, h].abs().T).amax(-1) * scale
                lse[s0 + i, hs] = torch.logsumexp(sc, -1)
                out[s0 + i, hs] = p @ Vs[:, h]
                spread[s0 + i, hs] = p @ Vs[:, h].abs()
    return out, lse, spread, reach
