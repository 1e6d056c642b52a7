"""Attention over drafted trees whose queries take so many CTAs that the keys stay in one share: one launch, no room for parts, with and without a workspace the same bits."""
import pytest
import torch
from gpu_helpers import dev
from test_gpu_attention_tree import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("starts,counts,nodes,n_q,n_kv", [([700], [256], 256, 20, 1), ([30, 600], [148, 100], 148, 64, 1), ([550], [75], 75, 64, 1)])
def test_one_share(cuda_lib, starts, counts, nodes, n_q, n_kv):
    from tenzo_b200 import kernels
    case = Case(nodes, starts, counts, nodes, n_q, n_kv)
    cache, start, a = case.arguments()
    q = dev(case.q)
    got = [kernels.attention_tree(q, cache, start, want_lse=True, workspace=w, shares=s, **a)
           for w, s in ((None, 0), (None, 1), (torch.empty(0, dtype=torch.uint8, device="cuda"), 0), (torch.empty(1 << 20, dtype=torch.uint8, device="cuda"), 0))]
    case.check(*got[0])
    for out, lse in got[1:]:
        assert torch.equal(out, got[0][0]) and torch.equal(lse, got[0][1])
    assert kernels.kv8_take_errors() == 0


def test_the_largest_number_of_heads(cuda_lib):
    """2^17 heads over one kv head: the call takes a few bytes of workspace, not tens of gigabytes."""
    from tenzo_b200 import kernels
    n_q = 1 << 17
    case = Case(5, [20], [2], 2, 20, 1, masked=False, rotated=False, spare=1000)
    cache, start, a = case.arguments()
    a["n_q"] = n_q
    q = dev(case.q).reshape(2, 20, 128)[:, torch.arange(n_q, device="cuda") % 20].reshape(2, n_q * 128)
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out, lse = kernels.attention_tree(q, cache, start, want_lse=True, max_len=900, **{k: v for k, v in a.items() if k != "max_len"})
    assert torch.cuda.max_memory_allocated() - before < q.numel() * 4 + lse.numel() * 4 + (16 << 20)
    for h in (0, 7, 19):
        assert bool((out.reshape(2, n_q, 128)[:, h::20] == out.reshape(2, n_q, 128)[:, h: h + 1]).all())
    case.check(out.reshape(2, n_q, 128)[:, :20].reshape(2, -1), lse[:, :20])
