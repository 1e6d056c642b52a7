"""Attention over drafted trees where one walk is so long that its accumulators are moved on though no reference changes, with the largest sums that codes and weights can make; and what a table entry out
of range leaves of the rows that would see its block."""
import numpy as np
import pytest
import kv8_reference as ref
from gpu_helpers import dev, host
from test_gpu_attention_tree import Case, check_weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("keys,nodes,n_q", [(32752, 1, 4), (70000, 1, 4), (40000, 7, 4), (33000, 12, 4), (40000, 16, 4)])
def test_long_walks(cuda_lib, keys, nodes, n_q):
    """Scores that do not grow: random ones, whose references stay for hundreds of tiles."""
    from tenzo_b200 import kernels
    case = Case(nodes, [keys], [nodes], nodes, n_q, 1, rotated=False, scale=0.2)
    cache, start, a = case.arguments()
    want = case.want()
    q = dev(case.q)
    for shares in (1, 2, 0):
        out, lse = kernels.attention_tree(q, cache, start, want_lse=True, shares=shares, **a)
        case.check(out, lse, want)
    check_weights(case, q, lse, cache, start, a, want)


@pytest.mark.parametrize("code", [127, -128])
@pytest.mark.parametrize("nodes", [1, 8, 12, 16])
def test_the_largest_sums(cuda_lib, nodes, code):
    """Values of one sign at the end of their range, and weights that are nearly 2^5 of the first tile's, which is as far as they go without a new reference: every output is the one value that there is."""
    from tenzo_b200 import kernels
    keys = 66000
    case = Case(nodes, [keys], [nodes], nodes, 4, 1, rotated=False, masked=False)
    b, o = case.c.at(0, np.arange(keys + nodes))
    case.q[:] = 1.0
    case.c.k[b, 0, 0, o] = 100
    rise = 4.98 * np.log(2)                                                     # of the argument, behind the first tile
    scale = np.where(np.arange(keys + nodes) < 128, 1.0, 1.0 + rise) * np.sqrt(128) / (100 * 128)
    case.c.sk[b, 0, 0, o] = scale
    case.c.sv[b, 0, 0, o] = np.float32(0.0312)                                  # just below a power of two: words with all bits in use
    case.c.v[b, 0, 0, o] = code
    cache, start, a = case.arguments()
    value = np.float64(np.float32(0.0312)) * code
    for shares in (1, 2, 0):
        out, lse = kernels.attention_tree(dev(case.q), cache, start, want_lse=True, shares=shares, **a)
        # weights are equal but for the first tile's, so their roundings (2^-27 of the largest each) are the sum's; sums of keys/128 numbers a thread in fp32, outputs moved on once in 256 tiles
        tol = abs(value) * (2.0 ** -26 + (keys / 128 + 16) * 2.0 ** -24)
        assert np.abs(host(out).astype(np.float64) - value).max() <= tol
        s = scale.astype(np.float32).astype(np.float64) * 100 * 128 / np.sqrt(128)
        for i in range(nodes):
            x = s[: keys + i + 1]
            assert np.abs(host(lse)[i] - (x.max() + np.log(np.exp(x - x.max()).sum()))).max() <= (keys / 128 + 64) * 2.0 ** -24
    assert kernels.kv8_take_errors() == 0


@pytest.mark.parametrize("nodes,start", [(9, 60), (1, 700), (40, 200), (20, 90)])
@pytest.mark.parametrize("shares", [0, 1, 3])
def test_a_block_that_is_none_is_left_out(cuda_lib, nodes, start, shares):
    """Rows come out as if its keys were not there, those of the tree among them, and with tiles in which nothing else is."""
    from tenzo_b200 import kernels
    for column in (0, 2, (start + nodes - 1) // 16):
        case = Case(nodes + start, [start], [nodes], nodes, 20, 5)
        cache, at, a = case.arguments()
        table = cache.block_table.clone()
        table[0, column] = -1 if column == 2 else case.c.n_blocks
        out, lse = kernels.attention_tree(dev(case.q), kernels.Kv8Cache(*cache[:4], table), at, want_lse=True, shares=shares, **a)
        assert kernels.kv8_take_errors() == 2
        gone = set(range(16 * column, 16 * column + 16))
        _, _, bound, lse_bound, _ = case.want()                                  # (fewer keys: a smaller bound; this one is let through)
        for i in range(nodes):
            places = np.array([t for t in list(range(start)) + sorted(start + j for j in case.sees[i]) if t not in gone], int)
            for h in range(5):
                key, value = (case.c.rows(x, 0, 0, h, start + nodes)[places] for x in "kv")
                x = ref.rotate(case.q[i].reshape(20, 128)[4 * h: 4 * h + 4], case.cos[case.pos[i]], case.sin[case.pos[i]])
                for g in range(4):
                    got, got_lse = host(out[i]).reshape(20, 128)[4 * h + g], float(lse[i, 4 * h + g])
                    if not len(places):
                        assert (got == 0).all() and got_lse == -np.inf
                        continue
                    s = key @ x[g] / np.sqrt(128)
                    e = np.exp(s - s.max())
                    r = slice((4 * h + g) * 128, (4 * h + g + 1) * 128)
                    assert (np.abs(got - e @ value / e.sum()) <= bound[i, r]).all()
                    assert abs(got_lse - s.max() - np.log(e.sum())) <= lse_bound[i, 4 * h + g] * (1 + abs(got_lse))
