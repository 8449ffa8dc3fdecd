"""How attention over a paged cache is cut over the grid (ae_b200/csrc/paged_plan.cuh) where the tensor-core
kernel's plan has to share the segments out along a line: more segments of one row tile than SMs, and more
sequences than threads plan.  Against 64 bits, with the tolerances of ``tests/test_gpu_paged.py``."""
import pytest
import torch

from tests.test_gpu_paged import BF, FP, call, compare, make_batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("D,dtype", [(128, BF), (64, FP)])
@pytest.mark.parametrize("Hq,n", [(16, 32), (32, 40)])
def test_more_segments_than_sms(Hq, n, D, dtype, bits):
    """24 trees x 8 key heads: 192 segments of 64 rows (one row tile of 128) and of 160 (one of 256)."""
    new = [n - b % 5 for b in range(24)]
    keys = [new[b] + (97 * b) % 700 for b in range(24)]
    d = make_batch(new, keys, Hq, 8, D, 16, dtype, bits, True, seed=21)
    out, lse = call(d)
    compare(d, out, lse)
    for _ in range(20):
        again, lse2 = call(d)
        assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("tree", [False, True], ids=["causal", "tree"])
@pytest.mark.parametrize("Hq", [16, 64])
def test_more_sequences_than_threads_plan(Hq, tree, bits):
    """200 sequences, of 6 tokens on average (48 and 192 rows of a key head), some of none and some of no context."""
    new = [(5 * b) % 13 for b in range(200)]
    keys = [new[b] + (31 * b) % 400 * (b % 3 > 0) for b in range(200)]
    d = make_batch(new, keys, Hq, 2, 128, 16, BF, bits, tree, seed=22)
    out, lse = call(d)
    compare(d, out, lse)
    for _ in range(20):
        again, lse2 = call(d)
        assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("tree", [False, True], ids=["causal", "tree"])
@pytest.mark.parametrize("Hq", [2, 8, 64])
def test_fewer_keys_than_new_tokens(Hq, tree, bits):
    """Sequences whose first new tokens have no key (a cut cache, a padded batch), beside whole ones, in every kernel:
    token i then sees the keys up to key i - (n - keys), and a tree's bits count from the same place."""
    new, keys = [60, 3, 40, 1, 17], [20, 3, 1, 0, 200]
    d = make_batch(new, keys, Hq, 2, 64, 16, FP, bits, tree, seed=23)
    out, lse = call(d)
    compare(d, out, lse)


def test_lengths_that_change_between_replays():
    """A captured call follows the lengths on the device: from one sequence that holds all tokens to tokens spread
    over 200, from no keys to many."""
    from ae_b200 import paged
    new, keys = [(3 * b) % 7 for b in range(200)], [300 - b for b in range(200)]
    d = make_batch(new, keys, 64, 2, 128, 16, BF, 16, False, seed=24)
    N = sum(new)
    lse = torch.zeros(N, 64, device="cuda")
    out = torch.zeros_like(d["q"])

    def step():
        paged.paged_attention(d["q"], d["k_cache"], d["v_cache"], d["block_table"], d["kv_lens"], d["q_starts"], out=out, lse=lse)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    whole, lens = d["q_starts"].clone(), d["kv_lens"].clone()
    for at in (0, 120, 199, None):
        if at is not None:
            d["q_starts"].copy_(torch.where(torch.arange(201, device="cuda") > at, N, 0))
            d["kv_lens"].copy_(torch.where(torch.arange(200, device="cuda") == at, lens, 0))
        else:
            d["q_starts"].copy_(whole)
            d["kv_lens"].copy_(lens)
        out.fill_(7.0)
        lse.fill_(7.0)
        graph.replay()
        compare(d, out, lse)
