"""Calls on trees one behind another with programmatic launches, of widths that cannot share an SM's tensor memory, give the bits of calls that wait for each other; one by one and captured."""
import pytest
import torch
from gpu_helpers import dev
from test_gpu_attention_tree import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("captured", [False, True])
def test_chains_of_unlike_widths(cuda_lib, captured):
    from tenzo_b200 import kernels
    cases = [Case(61 + i, [500, 90, 1200], [n, n, n], n, 4, 1) for i, n in enumerate((12, 1, 16, 4, 8))]     # 48, 16, 64, 16 and 32 queries a kv head
    sets = []
    for case in cases:
        cache, start, a = case.arguments()
        q = dev(case.q)
        out, lse = kernels.attention_tree(q, cache, start, want_lse=True, **a)
        weight = torch.zeros_like(dev(case.c.weight))
        kernels.kv8_weigh(q, lse, cache, weight, start, **a)
        sets.append((cache, start, a, q, out, lse, weight))
    torch.cuda.synchronize()

    def chain():
        got = []
        for turn in range(4):
            for i in range(len(sets)):
                cache, start, a, q, _, lse, weight = sets[(i * 2 + turn) % len(sets)]
                w = torch.zeros_like(weight)
                for _ in range(3):                                             # nothing but these kernels in between
                    kernels.kv8_weigh(q, lse, cache, w, start, use_pdl=True, **a)
                    again = kernels.attention_tree(q, cache, start, want_lse=True, use_pdl=True, **a)
                got.append(((i * 2 + turn) % len(sets), again, w))
            for i in (0, 1, 0, 2, 1, 2, 3, 0):
                cache, start, a, q, _, lse, weight = sets[i]
                got.append((i, kernels.attention_tree(q, cache, start, want_lse=True, use_pdl=True, **a), None))
        return got

    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = chain()
        for _ in range(5):
            graph.replay()
    else:
        got = chain()
    torch.cuda.synchronize()
    for i, (out, lse), w in got:
        assert torch.equal(out, sets[i][4]) and torch.equal(lse, sets[i][5])
        if w is not None:
            assert torch.allclose(w, 3 * sets[i][6], rtol=2.0 ** -22, atol=0)   # three additions, each rounded
    assert kernels.kv8_take_errors() == 0
