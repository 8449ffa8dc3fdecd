"""The status word of the paged cache's calls: what its codes raise (CPU), and the verify decoder's word (GPU)."""
import pytest
import torch

from ae_b200 import _native, build, paged


def test_codes_raise_once():
    build.build()
    word = torch.zeros(1, dtype=torch.int32)
    paged.check_status(word)
    for code, error in ((paged.BAD_PAGE, -10), (paged.TIMEOUT, -9)):
        word.fill_(code)
        with pytest.raises(_native.NativeError) as e:
            paged.check_status(word)
        assert e.value.code == error and int(word) == 0
        paged.check_status(word)


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["paged", "paged4"])
def test_decoder_reports_what_its_layers_recorded(cache):
    from ae_b200.verify import VerifyDecoder, random_tree
    from tests.test_gpu_verify_paged import config
    dec = VerifyDecoder(config(), batch=2, cache_len=70, max_draft=8, device="cuda", seed=1, cache=cache, page_size=16)
    tokens, parents = torch.zeros(2, 8, dtype=torch.int64, device="cuda"), random_tree(8, seed=2)
    good = dec.forward(tokens, parents)
    dec.check_status()
    page = int(dec.block_table[1, 2])
    dec.block_table[1, 2] = dec.block_table.numel()
    dec.forward(tokens, parents)
    dec.block_table[1, 2] = page
    with pytest.raises(_native.NativeError) as e:
        dec.check_status()
    assert e.value.code == -10
    assert torch.equal(dec.forward(tokens, parents), good)
    dec.check_status()
    slots = dec.slots
    dec.slots = slots + dec.block_table.numel() * 16
    dec.forward(tokens, parents)
    with pytest.raises(_native.NativeError):
        dec.check_status()


def test_dense_decoder_has_nothing_to_report():
    from ae_b200.verify import DecoderConfig, VerifyDecoder
    cfg = DecoderConfig(layers=1, H=64, I=64, E=2, k=1, heads=2, kv_heads=1, head_dim=64, vocab=10)
    VerifyDecoder(cfg, 1, 2, 2, "cpu").check_status()
