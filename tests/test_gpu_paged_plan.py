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
