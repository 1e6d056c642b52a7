"""The workspace of attention over drafted trees holds what a cut leaves: where a tree's queries take so many CTAs that its keys stay in one share, nothing is cut and next to nothing is needed, however many
queries there are."""
import pytest
from tenzo_b200 import kernels, load_library


@pytest.mark.parametrize("sequences,nodes,n_q,n_kv", [(1, 256, 20, 1), (1, 256, 1 << 17, 1), (64, 256, 1 << 17, 1), (3, 200, 64, 1), (2, 256, 40, 2), (7, 148, 64, 1)])
def test_one_share_needs_no_room_for_parts(sequences, nodes, n_q, n_kv):
    room = load_library().tenzo_cuda_attention_tree_workspace_bytes(sequences, nodes, n_q, n_kv, 0)
    assert 0 < room <= 8 * sequences * n_kv + 32 and room == kernels.attention_tree_workspace_bytes(sequences, nodes, n_q, n_kv)


@pytest.mark.parametrize("n_q", [1, 7, 20, 64, 1 << 17])
def test_some_megabytes_at_most(n_q):
    need = load_library().tenzo_cuda_attention_tree_workspace_bytes
    for nodes in (1, 2, 3, 8, 16, 31, 64, 100, 255, 256):
        assert 0 < need(1, nodes, n_q, 1, 0) < 24 << 20


def test_shares_that_are_asked_for_have_room():
    need = load_library().tenzo_cuda_attention_tree_workspace_bytes
    assert need(1, 256, 64, 1, 2) == 16 + 2 * 256 * 2 * 64 * 520
    assert need(1, 256, 64, 1, 1) >= 16
