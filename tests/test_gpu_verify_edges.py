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
