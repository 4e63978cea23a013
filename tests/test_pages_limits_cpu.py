"""The paged cache's and window attention's entry points at the largest sizes that they take, before anything is enqueued."""

from spec_mcts_b200._lib import lib
from test_pages_cpu import SHAPE, WORKSPACE, append, attn


def test_window_workspace_of_2_to_30_positions():
    """A query behind 2^30 - 1 keys, all of which are first keys as well, has CTAs share them as one behind half of them does."""
    need = lambda keys: lib.q40_attn_causal_window_workspace_bytes(1, 1, 1, 128, keys - 1, keys, keys)
    assert need(1 << 30) == need(1 << 29) == 16 * 130 * 4


def test_attention_of_2_to_29_keys():
    """Chunks of 8192 keys would be 65536 of them, one more than a grid has."""
    need = lambda keys: lib.q40_attn_pages_workspace_bytes(2, 4, 2, keys, 0, 0)
    row = 4 * 2 * 130 * 4                                     # two sequences, two kv heads, two heads each
    for keys in (65535 * 8192, 65535 * 8192 + 1, (1 << 29) - 1, 1 << 29):
        assert attn(L=keys, tstride=1 << 25) == WORKSPACE and need(keys) == 65535 * row
    assert need(1 << 28) == 32768 * row and attn(L=(1 << 29) + 1, tstride=1 << 26) == SHAPE


def test_append_refuses_8_bit_pages_above_2_to_26():
    """One CTA codes a page's earlier rows anew, 2^27 of them in 2^31 pieces."""
    for kind in (1, 2):
        assert append(ps=1 << 27, P=1 << 27, kind=kind, B=0, T=0) == SHAPE
        assert append(ps=(1 << 26) + 1, P=(1 << 26) + 1, kind=kind, B=0, T=0) == SHAPE
        assert append(ps=1 << 26, P=1 << 26, kind=kind, B=0, T=0) == 0
    assert append(ps=1 << 29, P=1 << 29, kind=0, B=0, T=0) == 0
