"""The operators of a drafted-token step on batches that are wrong, very uneven or mostly masked: what
test_gpu_draft_ops.py does not reach.  Its references and tolerances are used here too."""
import numpy as np
import pytest

from helpers import nfm
from test_gpu_draft_ops import check_attention, ints, make_cache

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
m = nfm()


def best_us(f, n=5):
    """The shortest of n passes, by events."""
    times = []
    for _ in range(n + 1):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        f()
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b) * 1e3)
    return min(times[1:])


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("n", [1, 300])
def test_refused_sequences_among_others(kind, n):
    """Several refused sequences of n rows become NaN in every row and head; the others and the rows behind stay as they are
    without them.  (Contexts of a tile: no item is in parts, so the others' sums have the same order.)"""
    rng = np.random.default_rng(n)
    nq, nkv, dim = 12, 2, 128
    c, _, _ = make_cache(rng, kind, 5, nkv, 400, dim)
    rows = [2, n, 0, n, 3]
    start = np.concatenate([[0], np.cumsum(rows)])
    total = int(start[-1])
    q = torch.from_numpy(rng.standard_normal((total + 2, nq, dim)).astype(np.float32)).bfloat16().cuda()
    work = torch.empty(m.tree_attention_workspace(dim), dtype=torch.uint8, device="cuda")
    good = [10, 20, 0, 30, 50]
    want = torch.full_like(q, 5.0)
    m.tree_attention(c, q, ints(start), ints(good), want, work)
    for prefix, seq in (([10, -1, 7, 401 - n, 50], None), ([10, 20, -9, 30, 50], [0, 5, 9, -1, 4])):
        out, status = torch.full_like(q, 5.0), ints([0])
        m.tree_attention(c, q, ints(start), ints(prefix), out, work, cache_seq=None if seq is None else ints(seq), status=status)
        assert status.item() != 0
        assert out[2:2 + n].isnan().all() and out[2 + n:2 + 2 * n].isnan().all()
        for r in (slice(0, 2), slice(2 + 2 * n, total)):
            assert (out[r].float() - want[r].float()).abs().max() <= 2.0 ** -7 * want[r].float().abs().max()
        assert torch.all(out[total:] == 5.0)


@pytest.mark.parametrize("rows", [1, 512])
def test_a_refused_sequence_takes_no_longer_than_a_good_one(rows):
    """Its rows are filled by the whole grid; one thread that fills them takes 100 us a row of 32 heads of 128."""
    nq, nkv, dim = 32, 4, 128
    c, _, _ = make_cache(np.random.default_rng(2), "e4m3", 2, nkv, 1000, dim)
    q = torch.zeros(rows + 1, nq, dim, dtype=torch.bfloat16, device="cuda")
    out, work = torch.zeros_like(q), torch.empty(m.tree_attention_workspace(dim), dtype=torch.uint8, device="cuda")
    start, good, bad = ints([0, rows, rows + 1]), ints([400, 999]), ints([-1, 999])
    fine = best_us(lambda: m.tree_attention(c, q, start, good, out, work))
    refused = best_us(lambda: m.tree_attention(c, q, start, bad, out, work))
    assert out[:rows].isnan().all()
    assert refused <= 2 * fine + 20, (refused, fine)
