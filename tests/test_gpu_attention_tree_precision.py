"""How good attention over drafted trees is where the numbers are of unlike sizes: values' scales far apart, keys that have most of the weight and small values, queries with single large dims. Against
64 bits, by the norm of each head's output.

The tolerance counts roundings. An argument of the exponential (s, natural units) is a product of four factors, each rounded once to fp32 (2^-24), minus a reference and plus a scale's logarithm, rounded once
as it is (w, in halvings), and the exponential is off by 2^-22: together d = 2^-24 (3 |s| + |w| + 4 + 4) at most, which moves a weight by itself and all others by way of the sum: 2 d, for the largest |s| and |w|
that matter. The query's fixed point adds half of 2^-29 of its largest number times the key's sum of magnitudes. A weight times its value's scale is rounded to 2^-26 of the largest such product that the
row sees; those errors are independent, 1/sqrt(12) of a step each, and six times their norm is let through."""
import numpy as np
import pytest
import torch
import kv8_reference as ref
from gpu_helpers import dev, host
from test_gpu_attention_tree import Case

pytestmark = pytest.mark.gpu


def want(case, s=0):
    """out [nodes, n_q, 128], lse, tolerances of the norms [nodes, n_q] and of lse, the weights [nodes, n_q, keys], and the bound d of their arguments; not rotated."""
    start, count, n_q, group = case.starts[s], case.counts[s], case.n_q, case.n_q // case.c.n_kv
    n = start + count
    out, lse, tol, lse_tol, weights, bound = np.zeros((count, n_q, 128)), np.zeros((count, n_q)), np.zeros((count, n_q)), np.zeros((count, n_q)), np.zeros((count, n_q, n)), np.zeros((count, n_q))
    b, o = case.c.at(s, np.arange(n))
    for h in range(case.c.n_kv):
        key, value = (case.c.rows(x, 0, s, h, n) for x in "kv")
        codes, scale = case.c.v[b, 0, h, o].astype(np.float64), case.c.sv[b, 0, h, o].astype(np.float64)
        for i in range(count):
            seen = np.array(list(range(start)) + sorted(start + j for j in case.sees[s * case.nodes + i] if j < count), int)
            for head in range(h * group, (h + 1) * group):
                x = case.q[s * case.nodes + i].reshape(n_q, 128)[head].astype(np.float64)
                arg = key[seen] @ x / np.sqrt(128)
                p = np.exp(arg - arg.max())
                lse[i, head] = arg.max() + np.log(p.sum())
                p /= p.sum()
                out[i, head] = p @ value[seen]
                heavy = p * scale[seen] > 1e-9 * (p * scale[seen]).max()
                spread = np.abs(np.log2(scale[seen][heavy] / scale[seen].max())).max()
                query = 2.0 ** -30 * np.abs(x).max() * np.abs(key[seen][heavy]).sum(-1).max() / np.sqrt(128)
                d = 2.0 ** -24 * (3 * np.abs(arg[heavy]).max() + np.ptp(arg[heavy]) * 1.4427 + spread + 8) + query
                step = 2.0 ** -26 * (p * scale[seen]).max()
                tol[i, head] = 2 * d * np.linalg.norm(out[i, head]) + 6 * step / np.sqrt(12) * np.linalg.norm(codes[seen])
                lse_tol[i, head] = 2 * d + (16 + len(seen) / 16) * 2.0 ** -24 + 4 * 2.0 ** -24 * (1 + abs(lse[i, head]))
                weights[i, head, seen], bound[i, head] = p, d
    return out, lse, tol, lse_tol, weights, bound


def check(case, shares=(0, 1, 3), rows=None):
    from tenzo_b200 import kernels
    cache, start, a = case.arguments()
    out, lse, tol, lse_tol, weights, bound = want(case)
    rows = slice(None) if rows is None else rows
    for n in shares:
        got, got_lse = kernels.attention_tree(dev(case.q), cache, start, want_lse=True, shares=n, **a)
        off = np.linalg.norm(host(got).astype(np.float64).reshape(-1, case.n_q, 128)[: len(out)] - out, axis=-1)
        print(f"shares {n}: error / norm {(off / np.linalg.norm(out, axis=-1))[rows].max():.2e}, / tolerance {(off / tol)[rows].max():.2f}")
        assert (off <= tol)[rows].all()
        assert (np.abs(host(got_lse)[: len(out)] - lse) <= lse_tol)[rows].all()
    weight = torch.zeros_like(dev(case.c.weight))
    kernels.kv8_weigh(dev(case.q), got_lse, cache, weight, start, **a)
    group = case.n_q // case.c.n_kv
    b, o = case.c.at(0, np.arange(weights.shape[2]))
    for h in range(case.c.n_kv):
        w = weights[:, h * group: (h + 1) * group]
        slack = (w * (2 * bound + lse_tol)[:, h * group: (h + 1) * group, None]).sum((0, 1)) + w.sum((0, 1)) * (16 + case.nodes * group / 8) * 2.0 ** -24
        assert (np.abs(host(weight)[b, 0, h, o] - w.sum((0, 1))) <= slack + 1e-30).all()
    assert kernels.kv8_take_errors() == 0


@pytest.mark.parametrize("factor", [2.0 ** 8, 2.0 ** 16, 2.0 ** 30])
@pytest.mark.parametrize("nodes,n_q,n_kv", [(12, 4, 1), (40, 6, 2), (64, 5, 5), (24, 2, 1)])
def test_a_sibling_of_large_values(cuda_lib, nodes, n_q, n_kv, factor):
    """A node whose values are far larger than all others' does not make the outputs of the rows coarser that do not see it."""
    case = Case(nodes, [700], [nodes], nodes, n_q, n_kv, rotated=False)
    b, o = case.c.at(0, 700 + nodes // 2)
    case.c.sv[b, 0, :, o] *= np.float32(factor)
    check(case, rows=[i for i in range(nodes) if nodes // 2 not in case.sees[i]])
    check(case)


@pytest.mark.parametrize("scale", [1e6, 3e38])
@pytest.mark.parametrize("nodes,n_q,n_kv", [(12, 4, 1), (24, 4, 2), (40, 6, 2), (64, 5, 5)])
def test_a_node_that_nobody_sees_has_no_part(cuda_lib, nodes, n_q, n_kv, scale):
    """Its row may hold anything: not a bit of the outputs changes."""
    from tenzo_b200 import kernels
    case = Case(nodes, [300], [nodes], nodes, n_q, n_kv, rotated=False)
    gone = nodes // 2
    case.sees = [s - {gone} | {0} for s in case.sees]
    got = []
    for value in (0.02, scale):
        b, o = case.c.at(0, 300 + gone)
        case.c.sv[b, 0, :, o] = case.c.sk[b, 0, :, o] = np.float32(value)
        cache, start, a = case.arguments()
        for shares in (0, 1, 2):
            got.append(kernels.attention_tree(dev(case.q), cache, start, want_lse=True, shares=shares, **a))
    for i in range(3):
        assert torch.equal(got[i][0], got[i + 3][0]) and torch.equal(got[i][1], got[i + 3][1])


@pytest.mark.parametrize("above,value", [(10, 0.01), (15, 0.001), (8, 100.0), (-15, 1000.0), (-25, 65536.0)])
@pytest.mark.parametrize("place", [0, 77, 2999])
@pytest.mark.parametrize("nodes,n_q", [(1, 4), (6, 4), (9, 8), (40, 4)])
def test_one_key_apart_from_all_others(cuda_lib, nodes, n_q, place, above, value):
    """A key that has most of the weight and small values, as the first token often has, and keys of little weight and large values."""
    case = Case(nodes + place, [3000], [nodes], nodes, n_q, 1, rotated=False, masked=False, scale=1.0)
    along = np.where(np.random.default_rng(5).random(128) < 0.5, -1, 1)
    case.q = (case.q.reshape(nodes, n_q, 128) + along).astype(np.float32).reshape(nodes, -1)
    b, o = case.c.at(0, place)
    case.c.k[b, 0, 0, o] = 100 * np.sign(above) * along
    case.c.sk[b, 0, 0, o] = np.float32(abs(above) / 100 / np.sqrt(128))
    case.c.sv[b, 0, 0, o] *= np.float32(value)
    check(case)


@pytest.mark.parametrize("dim,times,there", [(3, 100, 0.05), (64, 1000, 0.0), (127, 30, 1.0), (0, 1e5, 0.0)])
@pytest.mark.parametrize("nodes,n_q,n_kv", [(1, 4, 1), (9, 8, 2), (33, 6, 3), (64, 4, 1)])
def test_queries_with_one_large_dim(cuda_lib, nodes, n_q, n_kv, dim, times, there):
    """Where the keys are small, the other dims decide."""
    case = Case(nodes + dim, [2000], [nodes], nodes, n_q, n_kv, rotated=False, scale=1.0)
    q = case.q.reshape(nodes, n_q, 128)
    q[:, :, dim] = times * np.sign(q[:, :, dim])
    case.c.k[..., dim] = np.rint(case.c.k[..., dim] * there)
    check(case)


@pytest.mark.parametrize("step", [0.02, 0.5, 6.0])
def test_growing_scores_and_scales(cuda_lib, step):
    """The largest argument moves on from tile to tile, values' scales grow or fall meanwhile."""
    for ratio in (1.5, 1 / 1.5):
        case = Case(7, [1300], [16], 16, 20, 5, rotated=False, masked=False)
        b, o = case.c.at(0, np.arange(1316))
        case.c.k[b, 0, :, o] = np.sign(case.q[3].reshape(5, 4, 128)[:, 0]).astype(np.int8) * 20
        case.c.sk[b, 0, :, o] = (0.02 * step * (1 + np.arange(1316) // 100) * (1 + 0.01 * np.random.default_rng(3).random(1316)))[:, None]
        case.c.sv[b, 0, :, o] = (0.001 * ratio ** (np.arange(1316) // 90))[:, None]
        check(case)


def test_scales_of_zero(cuda_lib):
    """Values of nothing take their share of the weight; rows that see only such are zeros."""
    case = Case(9, [500], [20], 20, 4, 1, rotated=False)
    b, o = case.c.at(0, np.arange(500))
    case.c.sv[b[:200], 0, :, o[:200]] = 0
    case.c.sv[b[333], 0, :, o[333]] = 0
    from tenzo_b200 import kernels
    cache, start, a = case.arguments()
    for shares in (0, 1, 4):
        out, lse = kernels.attention_tree(dev(case.q), cache, start, want_lse=True, shares=shares, **a)
        case.check(out, lse)
    case.c.sv[b, 0, :, o] = 0
    case.sees = [set() for _ in range(20)]
    cache, start, a = case.arguments()
    out, lse = kernels.attention_tree(dev(case.q), cache, start, want_lse=True, **a)
    assert bool((out == 0).all()) and bool(torch.isfinite(lse).all())
    case.check(out, lse)
