"""The paged cache's and window attention's entry points at the largest sizes that they take, before anything is enqueued."""

from spec_mcts_b200._lib import lib


def test_window_workspace_of_2_to_30_positions():
    """A query behind 2^30 - 1 keys, all of which are first keys as well, has CTAs share them as one behind half of them does."""
    need = lambda keys: lib.q40_attn_causal_window_workspace_bytes(1, 1, 1, 128, keys - 1, keys, keys)
    assert need(1 << 30) == need(1 << 29) == 16 * 130 * 4
