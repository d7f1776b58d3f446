"""The operators of a drafted-token step on batches that are wrong, very uneven or mostly masked: what
test_gpu_draft_ops.py does not reach.  Its references and tolerances are used here too."""
import numpy as np
import pytest

from helpers import nfm
from test_gpu_draft_ops import check_attention, check_logprobs, exact_attention, ints, logits, make_cache, tree_words

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


def test_one_refused_sequence_of_many():
    """4,096 sequences of a row: one that is refused costs the others a look at every place, not one after another (1.0 ms
    where the call takes 0.44)."""
    nq, nkv, dim, batch = 32, 4, 128, 4096
    c, _, _ = make_cache(np.random.default_rng(3), "e4m3", 16, nkv, 512, dim)
    q = torch.ones(batch, nq, dim, dtype=torch.bfloat16, device="cuda")
    out, work = torch.zeros_like(q), torch.empty(m.tree_attention_workspace(dim), dtype=torch.uint8, device="cuda")
    start, seq, prefix = ints(range(batch + 1)), ints([i % 16 for i in range(batch)]), ints([200] * batch)
    fine = best_us(lambda: m.tree_attention(c, q, start, prefix, out, work, cache_seq=seq))
    assert not out.isnan().any()
    prefix[[0, 300, 4095]] = ints([-1, 512, 2 ** 31 - 1])
    refused = best_us(lambda: m.tree_attention(c, q, start, prefix, out, work, cache_seq=seq))
    bad = out.isnan().flatten(1)
    assert bad[[0, 300, 4095]].all() and bad.any(1).sum() == 3
    assert refused <= 1.5 * fine + 20, (refused, fine)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("singles, chunk", [(40, 200), (40, 100), (70, 100), (150, 60), (3, 300)])
def test_attention_of_a_chunk_among_single_rows(kind, singles, chunk):
    """One long chunk among decoding sequences, on both sides of the average that chooses the kernel."""
    rng = np.random.default_rng(singles + chunk)
    rows, at = [1] * (singles + 1), int(rng.integers(singles + 1))
    rows[at] = chunk
    prefix = rng.integers(0, 300, singles + 1).tolist()
    check_attention(chunk, rows, prefix, 8, 1, 64, kind, seq=rng.permutation(singles + 1).tolist(), context=300 + chunk)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_attention_of_a_batch_with_many_empty_places(kind):
    """A batch of fixed places of which few hold rows."""
    rows = [0] * 200
    rows[0], rows[77], rows[78], rows[199] = 1, 9, 1, 2
    prefix = [5 * i for i in range(200)]
    check_attention(3, rows, prefix, 8, 2, 64, kind, seq=[i % 7 for i in range(200)], seqs=7, context=1000)


@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("vocab", [20000, 40001, 151552])
def test_logprobs_of_masked_rows_over_several_ctas(wide, vocab):
    """Rows of which a grammar leaves a few tokens, and rows without a distribution, where several CTAs share a row: the top
    tokens go on with -infinity and then NaN, the lower index first."""
    rng = np.random.default_rng(vocab)
    x = logits(rng, 8, vocab, wide, pad=3)
    inf = float("inf")
    for r, left in enumerate((1, 3, 20, 33)):
        keep = torch.from_numpy(rng.choice(vocab, left, replace=False)).cuda()
        old = x[r, keep].clone()
        x[r] = -inf
        x[r, keep] = old
    x[4] = -inf
    x[5, vocab // 2:] = float("nan")
    x[6] = float("nan")
    x[7, :-1] = -inf
    target = torch.from_numpy(rng.integers(0, vocab, 8)).int().cuda()
    target[0] = int(x[0].float().argmax())
    for rows in (8, 1):  # eight and fewer CTAs a row
        for top in (32, 5, 1):
            check_logprobs(x[:rows], target[:rows], top)


def test_what_is_missing_is_refused_by_name():
    """None, a number or a list in a tensor's place is refused as the binding refuses other arguments."""
    c, _, _ = make_cache(np.random.default_rng(1), "bf16", 2, 1, 8, 64)
    q = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    w = torch.empty(m.tree_attention_workspace(64), dtype=torch.uint8, device="cuda")
    s, p, lg, f = ints([0, 1, 2]), ints([0, 0]), torch.zeros(2, 9, device="cuda"), torch.zeros(2, device="cuda")
    for word, call in (("workspace", lambda: m.tree_attention(c, q, s, p, q, None)), ("workspace", lambda: m.tree_attention(c, q, s, p, q, 5)),
                       ("q ", lambda: m.tree_attention(c, None, s, p, q, w)), ("row_start", lambda: m.tree_attention(c, q, [0, 2], p, q, w)),
                       ("prefix", lambda: m.tree_attention(c, q, s, None, q, w)), ("output", lambda: m.tree_attention(c, q, s, p, None, w)),
                       ("workspace", lambda: m.token_logprobs(lg, None, None, f, None, None, None)),
                       ("logits", lambda: m.token_logprobs(None, None, None, f, None, None, w)),
                       ("qkv", lambda: m.kv_write(c, m.Rope(64), None, 2, p, q)),
                       ("position", lambda: m.kv_write(c, m.Rope(64), torch.zeros(2, 256, device="cuda"), 2, None, q)),
                       ("path", lambda: m.kv_accept(m.KvCaches([c]), p, None, p)),
                       ("null", lambda: m.kv_accept(m.KvCaches([c]), p, p.view(2, 1), None))):
        with pytest.raises(m.NfError, match=word):
            call()
    m.tree_attention(c, q, s, p, torch.empty_like(q), w.view(-1, 64))  # a workspace of any shape will do


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("mask", [None, "any", "tree"])
@pytest.mark.parametrize("rows", [[200] + [1] * 150, [3, 150, 70], [7, 2, 9]])
def test_values_that_are_not_finite_in_a_long_sequence(kind, dim, mask, rows):
    """A NaN and an infinity in new rows' values reach the rows that see them, in every kernel, and take no row that does
    not; looking for those rows takes a small part of a call (65 ms where each thread looks for itself)."""
    rng = np.random.default_rng(len(rows) + dim)
    nq, nkv = 8, 1
    long, n = int(np.argmax(rows)), max(rows)
    prefix = rng.integers(0, 200, len(rows)).tolist()
    c, k, v = make_cache(rng, kind, len(rows), nkv, 450, dim)
    words = (n + 63) // 64
    start = np.concatenate([[0], np.cumsum(rows)])
    pairs = [tree_words(rng, r, words, mask) for r in rows] if mask else None
    bits = torch.from_numpy(np.concatenate([p[0] for p in pairs])).cuda() if mask else None
    q = torch.from_numpy(rng.standard_normal((int(start[-1]), nq, dim)).astype(np.float32)).bfloat16()
    out, work = torch.empty_like(q, device="cuda"), torch.empty(m.tree_attention_workspace(dim), dtype=torch.uint8, device="cuda")
    args = (c, q.cuda(), ints(start), ints(prefix), out, work)
    fine = best_us(lambda: m.tree_attention(*args, mask=bits))
    bad_rows = sorted({n - 1, n // 2})
    for i, j in enumerate(bad_rows):
        at = (long, 0, prefix[long] + j, 5 + 20 * i)
        if kind == "bf16":
            c.tensors[1][at] = float("nan") if i else float("inf")
        elif i:
            c.tensors[1].view(torch.uint8)[at] = 0xff
        else:
            c.tensors[3][at[:3]] = float("inf")
    took = best_us(lambda: m.tree_attention(*args, mask=bits))
    got = out.double().cpu().numpy()
    qd = q.double().numpy()
    for r in range(n):
        vis = np.ones(prefix[long] + n, bool)
        vis[prefix[long]:] = np.arange(n) <= r if mask is None else pairs[long][1][r][:n]
        mine = got[start[long] + r]
        if vis[prefix[long]:][bad_rows].any():
            assert np.isnan(mine).all(), r
        else:
            want, tol = exact_attention(qd[start[long] + r], k[long, 0, :len(vis)], v[long, 0, :len(vis)], vis, dim ** -0.5)
            assert np.all(np.abs(mine - want) <= tol), r
    rest = np.ones(len(got), bool)
    rest[start[long]:start[long + 1]] = False
    assert not np.isnan(got[rest]).any()
    assert took <= 4 * fine + 50, (took, fine)
