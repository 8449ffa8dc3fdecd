"""The verify-step decoder over paged caches (ae_b200/verify.py, cache="paged" / "paged4"): two layers
against the dense decoder of the same seed, and the attention half of a layer against 64 bits over the
cache that it left behind, for one draft token up to a tree of 40."""
import pytest
import torch

from tests import paged_reference as ref

pytestmark = pytest.mark.gpu


def config(heads=4, kv_heads=2):
    from ae_b200.verify import DecoderConfig
    return DecoderConfig(layers=2, H=512, I=256, E=8, k=2, heads=heads, kv_heads=kv_heads, head_dim=128, vocab=1000)


@pytest.mark.parametrize("n,page_size", [(32, 64), (1, 16), (40, 8)])
def test_paged_decoder_matches_the_dense_one(n, page_size):
    """Bar: relative L2 of the logits <= 2e-2 after two bf16 layers, as for the library's MoE block."""
    from ae_b200.verify import VerifyDecoder, random_tree
    parents = random_tree(n, seed=2)
    g = torch.Generator(device="cuda").manual_seed(1)
    tokens = torch.randint(0, 1000, (2, n), generator=g, device="cuda")
    make = lambda **kw: VerifyDecoder(config(), batch=2, cache_len=70, max_draft=40, device="cuda", seed=7, **kw)  # noqa: E731
    a = make(cache="paged", page_size=page_size).forward(tokens, parents)
    b = make().forward(tokens, parents)
    assert float((a.float() - b.float()).norm() / b.float().norm()) <= 2e-2


@pytest.mark.parametrize("cache", ["paged", "paged4"])
@pytest.mark.parametrize("n,heads", [(1, 4), (12, 8), (40, 16)])
def test_attention_half_against_64_bits(cache, n, heads):
    """Relative L2 <= 1e-2: the output is rounded to bf16 before the projection (2^-9 of itself, rms), the
    weights p, the values and, for many rows over 4 bits, the keys as much again (0.2 % each), and the
    projection's result once."""
    from ae_b200.verify import VerifyDecoder, random_tree
    cfg = config(heads, 2)
    dec = VerifyDecoder(cfg, batch=3, cache_len=200, max_draft=40, device="cuda", seed=3, cache=cache, page_size=32)
    parents = random_tree(n, seed=5)
    step = dec._paged_step(parents)
    h = torch.randn(3, n, cfg.H, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").bfloat16()
    out = dec._paged_attention(0, h, step)
    x = (h @ dec.layers[0]["wqkv"].t()).view(3 * n, heads + 4, 128)
    q = ref.rotate(x[:, :heads].double(), step["positions"], dec.inv_freq, False, 1.0).bfloat16()
    k = ref.rotate(x[:, heads:heads + 2].double(), step["positions"], dec.inv_freq, False, 1.0)
    kc, vc = dec.k_cache[0], dec.v_cache[0]
    page, at = step["slots"] // 32, step["slots"] % 32
    for c, want in ((kc, k), (vc, x[:, heads + 2:].double())):
        got = c[page, :, at].double() if cache == "paged" else ref.values(c[page, :, at], 128, torch.bfloat16)
        # 4 bits: half a step of a 15th of the group's range, 4 to 5 sigma
        assert float((got - want).norm() / want.norm()) <= (3e-3 if cache == "paged" else 0.11)
    o, _, _, _ = ref.attention(q, kc, vc, dec.block_table, step["kv_lens"], step["q_starts"], step["tree"])
    want = o.reshape(3, n, -1) @ dec.layers[0]["wo"].double().t()
    assert float((out.double() - want).norm() / want.norm()) <= 1e-2
