"""The decoder stack's step over several rows of a sequence on the batches
that a server makes by accident or on purpose: sequences that do not fit,
tokens and row starts outside, padded rows, several captured steps.

Caches are compared by the places that changed, bit for bit.  Hidden states
of the same rows in another batch take the same arithmetic up to the order of
F32 sums and are held to the tolerances of test_gpu_stack_verify.py."""
import numpy as np
import pytest

from helpers import nfm, workload
from test_gpu_stack_verify import CFG, close, ints, make_stack, model  # noqa: F401 (model is a fixture)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
m, wl = nfm(), workload()
H, V, L = CFG["hidden"], CFG["vocab"], 64


class DeviceBytes:
    """A span of device memory, for torch.as_tensor."""

    def __init__(self, ptr, n):
        self.__cuda_array_interface__ = dict(shape=(n,), typestr="|u1", data=(ptr, False), version=3)


def caches(st):
    """Copies of every layer's caches (codes and scales) as bytes."""
    out = []
    for layer in range(CFG["layers"]):
        d = st.kv_desc(layer)
        rows = d.seqs * d.kv_heads * d.max_context
        for ptr, n in ((d.k, rows * d.head_dim * (1 if d.kind == m.KV_E4M3 else 2)),
                       (d.v, rows * d.head_dim * (1 if d.kind == m.KV_E4M3 else 2)), (d.k_scale, 4 * rows), (d.v_scale, 4 * rows)):
            if ptr:
                out.append(torch.as_tensor(DeviceBytes(ptr, n), device="cuda").clone())
    return out


def changed(st, before):
    """Which (sequence, position) pairs of any layer's caches differ from their copies."""
    d = st.kv_desc(0)
    out = torch.zeros(d.seqs, d.max_context, dtype=torch.bool, device="cuda")
    for a, b in zip(before, caches(st)):
        out |= (a != b).view(d.seqs, d.kv_heads, d.max_context, -1).any(-1).any(1)
    return {(i, p) for i, p in out.nonzero().tolist()}


def step(st, tokens, start, prefix, depth=None, rows=None, sync=True):
    rows = len(tokens) if rows is None else rows
    fin = torch.full((rows, H), 3.0, dtype=torch.float32, device="cuda")
    nxt = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    st.verify(ints(tokens), ints(start), ints(prefix), rows, nxt, fin, depth=None if depth is None else ints(depth))
    if sync:
        st.sync()
    return fin, nxt


@pytest.mark.parametrize("kv", ["e4m3", "bf16"])
@pytest.mark.parametrize("what", ["prefix", "token"])
def test_the_other_sequences_go_on(model, kv, what):  # noqa: F811
    """A sequence that does not fit, or a token outside the vocabulary, becomes NaN and is reported; the sequences beside it
    get what they get without it."""
    tokens = np.random.default_rng(1).integers(0, V, 5)
    start = [0, 2, 3, 5]
    st = make_stack(model, 8, L, kv)
    st.fill_kv(3)
    fin, _ = step(st, tokens, start, [10, 5, 20])
    wrong = tokens.copy()
    if what == "token":
        wrong[2] = V
    st.fill_kv(3)
    got, _ = step(st, wrong, start, [10, L if what == "prefix" else 5, 20], sync=False)
    with pytest.raises(m.NfError, match="outside the cache"):
        st.sync()
    assert got[2].isnan().all()
    close(got[:2], fin[:2], "the sequence before")
    close(got[3:], fin[3:], "the sequence behind")
    st.sync()  # reported once, and nothing else is left to report
    st.close()


def test_decode_over_e4m3_caches_goes_on(model):  # noqa: F811
    tokens = np.random.default_rng(2).integers(0, V, 3)
    st = make_stack(model, 4, L, "e4m3")

    def decode(tok, pos):
        st.fill_kv(3)
        fin, nxt = torch.empty(3, H, device="cuda"), torch.empty(3, dtype=torch.int32, device="cuda")
        st.decode(ints(tok), ints(pos), 3, nxt, fin)
        return fin

    fin = decode(tokens, [10, 5, 20])
    st.sync()
    for tok, pos in ((tokens, [10, L, 20]), (tokens, [10, -1, 20]), ([tokens[0], -1, tokens[2]], [10, 5, 20])):
        got = decode(tok, pos)
        with pytest.raises(m.NfError, match="outside the cache"):
            st.sync()
        assert got[1].isnan().all()
        close(got[[0, 2]], fin[[0, 2]], "beside it")
    st.close()


@pytest.mark.parametrize("kv", ["e4m3", "bf16"])
def test_a_step_behind_a_refused_path(model, kv):  # noqa: F811
    """A path that is refused is reported by the next sync, and spoils no step before it."""
    tokens = np.random.default_rng(3).integers(0, V, 3)
    st = make_stack(model, 8, L, kv)
    st.fill_kv(3)
    fin, _ = step(st, tokens, [0, 3], [10])
    st.fill_kv(3)
    st.accept(ints([10]), ints([[3, 2]]), ints([2]))  # does not rise
    got, _ = step(st, tokens, [0, 3], [10], sync=False)
    with pytest.raises(m.NfError, match="outside the cache"):
        st.sync()
    close(got, fin, "behind a refused path")
    st.close()


@pytest.mark.parametrize("kv", ["e4m3", "bf16"])
@pytest.mark.parametrize("prefix, depth", [
    (-1, None), (-2, None), (-(2 ** 31), None), (L - 1, None), (L - 2, None), (L, None), (2 ** 31 - 1, None),
    (5, [0, -6, 1]), (5, [0, 1, 2 ** 31 - 1])])
def test_a_refused_sequence_writes_nothing(model, kv, prefix, depth):  # noqa: F811
    """A sequence of three rows whose prefix, rows or positions lie outside changes no cache, becomes NaN and is reported;
    the sequences beside it get what they get beside a sequence that fits."""
    tokens = np.random.default_rng(1).integers(0, V, 7)
    start = [0, 2, 5, 7]
    st = make_stack(model, 8, L, kv)
    st.fill_kv(3)
    fin, _ = step(st, tokens, start, [10, 5, 20], depth=None if depth is None else [0, 1, 0, 1, 2, 0, 1])
    st.fill_kv(3)
    before = caches(st)
    got, _ = step(st, tokens, start, [10, prefix, 20], depth=None if depth is None else [0, 1] + depth + [0, 1], sync=False)
    with pytest.raises(m.NfError, match="outside the cache"):
        st.sync()
    assert changed(st, before) == {(0, 10), (0, 11), (2, 20), (2, 21)}
    assert got[2:5].isnan().all()
    close(got[:2], fin[:2], "the sequence before")
    close(got[5:], fin[5:], "the sequence behind")
    st.close()


@pytest.mark.parametrize("kv", ["e4m3", "bf16"])
@pytest.mark.parametrize("start", [[-3, 3, 5], [-(2 ** 31), 3, 5], [0, 3, 99], [-1, 3, 2 ** 31 - 1]])
def test_row_starts_outside_are_clamped(model, kv, start):  # noqa: F811
    """Row starts below 0 and behind the rows count as 0 and as the number of rows, in the caches as in the attention."""
    tokens = np.random.default_rng(2).integers(0, V, 5)
    st = make_stack(model, 8, L, kv)
    st.fill_kv(4)
    fin, _ = step(st, tokens, [0, 3, 5], [10, 20])
    st.fill_kv(4)
    before = caches(st)
    got, _ = step(st, tokens, start, [10, 20])
    assert changed(st, before) == {(0, 10), (0, 11), (0, 12), (1, 20), (1, 21)}
    close(got, fin, "clamped")
    st.close()


def test_logprobs_of_replayed_steps(model):  # noqa: F811
    """Log-probabilities of a replayed step, whichever step was enqueued or captured since."""
    tokens = np.random.default_rng(5).integers(0, V, 6)
    st = make_stack(model, 8, L, "e4m3")
    args = [(ints(tokens[:n]), ints([0, n]), ints([10]), n, torch.empty(n, dtype=torch.int32, device="cuda"),
             torch.empty(n, H, device="cuda")) for n in (6, 2)]

    def logprobs():
        lp = torch.zeros(6, device="cuda")
        st.logprobs(6, ints([7] * 6), lp)
        st.sync()
        return lp

    def fresh():
        st.fill_kv(3)
        st.verify(*args[0])

    fresh()
    want = logprobs()
    s, graphs = torch.cuda.Stream(), []
    fresh()  # an eager step of 6 rows, then captures that do not run
    st.sync()
    for a in args:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=s):
            st.verify(*a, stream=torch.cuda.current_stream().cuda_stream)
    assert torch.equal(logprobs(), want)
    for i in (1, 0):  # the larger step is replayed last
        st.fill_kv(3)
        graphs[i].replay()
    assert torch.equal(logprobs(), want)
    with pytest.raises(m.NfError, match="rows"):
        st.logprobs(7, ints([7] * 7), torch.zeros(7, device="cuda"))
    st.close()


@pytest.mark.parametrize("kv", ["e4m3", "bf16"])
def test_padded_rows_need_no_token(model, kv):  # noqa: F811
    """Rows behind the last sequence (and in front of the first) may hold any token: nothing is reported, nothing written,
    and the others' results stand."""
    tokens = np.random.default_rng(6).integers(0, V, 3)
    st = make_stack(model, 8, L, kv)
    st.fill_kv(3)
    fin, _ = step(st, tokens, [0, 1, 3], [10, 20])
    for before, behind in ((0, 3), (2, 0), (1, 2)):
        st.fill_kv(3)
        old = caches(st)
        got, _ = step(st, [-1] * before + list(tokens) + [V, -1, 2 ** 31 - 1][:behind], [before, before + 1, before + 3], [10, 20])
        assert changed(st, old) == {(0, 10), (1, 20), (1, 21)}
        close(got[before:before + 3], fin, "beside padding")
    st.close()


def test_a_step_after_a_fill_without_memory(model):  # noqa: F811
    """An E4M3 cache is filled through a buffer of BF16 rows.  Without memory for that the call fails, and the next step
    does not."""
    context = 1 << 17
    st = make_stack(model, 8, context, "e4m3")
    need = 2 * 8 * context * CFG["kv_heads"] * 128
    torch.cuda.empty_cache()
    hold = torch.empty(torch.cuda.mem_get_info()[0] - need // 2, dtype=torch.uint8, device="cuda")
    with pytest.raises(m.NfError, match="memory"):
        st.fill_kv(3)
    del hold
    torch.cuda.empty_cache()
    fin, _ = step(st, [1, 2, 3], [0, 1, 3], [0, 0])
    assert not fin.isnan().any()
    st.close()
