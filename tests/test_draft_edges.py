"""What the operators of a drafted-token step refuse before any CUDA call, beyond test_draft_ops.py (on the CPU)."""
import pytest

from helpers import nfm
from test_draft_ops import cache, call_accept, message

m = nfm()


@pytest.mark.parametrize("heads, dim, kind", [(1 << 28, 64, m.KV_E4M3), ((1 << 31) - 1, 128, m.KV_BF16), (1 << 27, 128, m.KV_E4M3)])
def test_accept_refuses_more_pieces_than_32_bits_count(heads, dim, kind):
    """A thread moves 16 bytes of a row of K or V: heads x 2 x (dim / 8 + 1) of them at most."""
    scales = {} if kind == m.KV_E4M3 else dict(k_scale=None, v_scale=None)
    assert call_accept([cache(seqs=1, kv_heads=heads, head_dim=dim, kind=kind, **scales)], batch=1, max_path=1) == 10
    assert "2^31" in message()


def test_accept_takes_many_heads():
    assert call_accept([cache(seqs=1, kv_heads=1 << 24)]) == 0
