"""Attention of drafted trees over the INT8 caches, and the weights that cached tokens receive, against 64 bits. What lies in places that nobody sees is NaN in the
scales and anything in the codes."""
import numpy as np
import pytest
import torch
import kv8_reference as ref
from gpu_helpers import dev, host

pytestmark = pytest.mark.gpu


def parents(rng, n):
    return [-1] + [max(0, i - 1 - int(rng.integers(0, 4))) for i in range(1, n)]


class Case:
    def __init__(self, seed, starts, counts, nodes, n_q, n_kv, *, slots=16, layers=1, layer=0, masked=True, rotated=True, scale=1.5, spare=0):
        rng = self.rng = np.random.default_rng(seed)
        self.starts, self.counts, self.nodes, self.n_q, self.layer, self.masked, self.rotated = starts, counts, nodes, n_q, layer, masked, rotated
        n = len(starts)
        self.max_len = max(s + nodes for s in starts)
        self.c = ref.Caches(rng, n, (self.max_len + spare + slots - 1) // slots, layers, n_kv, slots)
        for s in range(n):
            self.c.fill(rng, s, range(max(0, starts[s] + counts[s])))
        self.q = (scale * rng.standard_normal((n * nodes, n_q * 128))).astype(np.float32)
        self.words = (nodes + 31) // 32
        self.sees = []
        for _ in range(n):
            self.sees += ref.ancestors(parents(rng, nodes)) if masked else [set(range(i + 1)) for i in range(nodes)]
        self.pos = rng.integers(0, self.max_len + 40, n * nodes).astype(np.int32)
        self.cos, self.sin = ref.rope(self.max_len + 40)

    def arguments(self):
        from tenzo_b200 import kernels
        c = self.c
        a = dict(layer=self.layer, n_q=self.n_q, nodes=self.nodes, count=dev(np.array(self.counts, np.int32)), max_len=self.max_len)
        if self.masked:
            m = ref.masks(self.sees, self.nodes, self.words).view(np.uint32)
            for i in range(len(m)):                                  # bits of nodes that are not there mean nothing
                n = self.counts[i // self.nodes]
                for j in range(n, 32 * self.words):
                    m[i, j // 32] |= np.uint32(1 << (j % 32))
            a["mask"] = dev(m.view(np.int32))
        if self.rotated:
            a |= dict(rope_pos=dev(self.pos), rope_cos=dev(self.cos), rope_sin=dev(self.sin))
        return kernels.Kv8Cache(dev(c.k), dev(c.v), dev(c.sk), dev(c.sv), dev(c.table)), dev(np.array(self.starts, np.int32)), a

    def want(self):
        out, lse, bound, lse_bound = np.zeros(self.q.shape), np.full((len(self.q), self.n_q), -np.inf), np.zeros(self.q.shape), np.zeros((len(self.q), self.n_q))
        weights = []
        for s, (start, count) in enumerate(zip(self.starts, self.counts)):
            r = slice(s * self.nodes, s * self.nodes + count)
            if start < 0 or count == 0:
                weights.append(None)
                continue
            turn = [(self.cos[p], self.sin[p]) for p in self.pos[r]] if self.rotated else None
            out[r], lse[r], bound[r], lse_bound[r], w = ref.tree(self.q[r], self.c, self.layer, self.n_q, (s, start), self.sees[r], turn)
            weights.append(w)
        return out, lse, bound, lse_bound, weights

    def check(self, out, lse, want=None):
        want_out, want_lse, bound, lse_bound, _ = want or self.want()
        out, lse = host(out).astype(np.float64), host(lse).astype(np.float64)
        assert np.isfinite(out).all() and np.array_equal(np.isneginf(lse), np.isneginf(want_lse))
        empty = np.repeat(np.isneginf(want_lse), 128, 1)
        assert (out[empty] == 0).all()
        assert (np.abs(out - want_out) <= bound).all(), (np.abs(out - want_out) / np.maximum(bound, 1e-30)).max()
        there = ~np.isneginf(want_lse)
        assert (np.abs(lse[there] - want_lse[there]) <= lse_bound[there]).all()
        norm = np.linalg.norm(want_out)
        assert norm == 0 or np.linalg.norm(out - want_out) <= 4e-6 * norm, np.linalg.norm(out - want_out) / norm      # (the bound above is the worst of all cases)


def check_weights(case, q, lse, cache, start, a, want):
    from tenzo_b200 import kernels
    weight = dev(case.c.weight)
    kernels.kv8_weigh(q, lse, cache, weight, start, **a)
    expect, slack = case.c.weight.astype(np.float64), np.zeros(case.c.weight.shape)
    for s, w in enumerate(want[4]):
        if w is None:
            continue
        b, o = case.c.at(s, np.arange(w.shape[1]))
        for h in range(case.c.n_kv):
            expect[b, case.layer, h, o] += w[h]
            # an exponential is off by what its argument is off; sums of up to nodes * group numbers and the old weight in fp32
            slack[b, case.layer, h, o] += w[h] * (2 * want[3].max() + (16 + case.nodes * case.n_q / case.c.n_kv / 8) * 2.0 ** -24)
    got = host(weight).astype(np.float64)
    assert (np.abs(got - expect) <= slack + 2.0 ** -23 * np.abs(expect)).all()
    assert np.array_equal(got[slack == 0], case.c.weight[slack == 0])                       # nothing else is touched
    assert kernels.kv8_take_errors() == 0


CASES = [
    # starts, counts, nodes, n_q, n_kv, further
    ([0], [1], 1, 1, 1, {}),
    ([5], [1], 1, 20, 5, {}),
    ([127, 128, 129], [1, 1, 1], 1, 20, 5, {}),
    ([1000], [8], 8, 20, 5, {}),
    ([0, 3, 600], [16, 16, 16], 16, 20, 5, {}),
    ([100, 260, 0, 33], [64, 1, 0, 40], 64, 20, 5, dict(layers=3, layer=1)),
    ([300, 17], [33, 20], 33, 7, 1, {}),
    ([120, 700], [27, 9], 27, 40, 5, {}),
    ([257], [256], 256, 8, 4, {}),
    ([90], [256], 256, 16, 16, {}),
    ([64, 1], [65, 2], 65, 12, 4, dict(slots=144)),
    ([200, 77], [5, 5], 5, 32, 2, dict(rotated=False)),
    ([333], [100], 100, 20, 5, dict(masked=False)),
    ([50, 400], [1, 1], 1, 6, 1, dict(masked=False, slots=416)),
    ([30, -1, 40], [3, 3, 2], 3, 64, 1, {}),
    ([64], [64], 64, 3, 1, dict(scale=8.0)),
    ([4000], [2], 2, 20, 5, dict(scale=0.01)),
    ([40], [256], 256, 32, 1, {}),                                            # 8192 queries of one kv head
]


@pytest.mark.parametrize("starts,counts,nodes,n_q,n_kv,further", CASES, ids=lambda x: "" if isinstance(x, dict) else str(x).replace(" ", ""))
def test_tree_and_weights(cuda_lib, starts, counts, nodes, n_q, n_kv, further):
    from tenzo_b200 import kernels
    case = Case(nodes * 100 + n_q, starts, counts, nodes, n_q, n_kv, **further)
    cache, start, a = case.arguments()
    q = dev(case.q)
    out, lse = kernels.attention_tree(q, cache, start, want_lse=True, **a)
    want = case.want()
    case.check(out, lse, want)
    check_weights(case, q, lse, cache, start, a, want)


@pytest.mark.parametrize("starts,nodes,n_q,n_kv", [([3300, 2700, 1999, 3500, 900, 3111, 2048], 70, 16, 8), ([5000, 4000, 6000, 2500], 1, 16, 16), ([2000, 3000, 1500, 2300], 100, 32, 16)])
def test_weights_of_long_shares(cuda_lib, starts, nodes, n_q, n_kv):
    """Enough keys that every CTA has many tiles, with queries of one pass, of five and of seven, the last of which take two walks."""
    from tenzo_b200 import kernels
    case = Case(nodes + 7, starts, [max(1, nodes - 3 * s) for s in range(len(starts))], nodes, n_q, n_kv)
    cache, start, a = case.arguments()
    q = dev(case.q)
    out, lse = kernels.attention_tree(q, cache, start, want_lse=True, **a)
    want = case.want()
    case.check(out, lse, want)
    check_weights(case, q, lse, cache, start, a, want)


@pytest.mark.parametrize("nodes,n_q", [(1, 20), (8, 20), (12, 20), (64, 20), (40, 40)])
@pytest.mark.parametrize("shares", [1, 2, 7, 13, 64, 1000])
def test_shares(cuda_lib, nodes, n_q, shares):
    """Cuts anywhere give what whole sequences do: several in one sequence's keys, several sequences between two, shares that nothing is left for."""
    from tenzo_b200 import kernels
    case = Case(shares + nodes, [1500, 100, -1, 640, 0, 3], [nodes, nodes, nodes, max(1, nodes - 3), nodes, 0], nodes, n_q, 5)
    cache, start, a = case.arguments()
    out, lse = kernels.attention_tree(dev(case.q), cache, start, want_lse=True, shares=shares, **a)
    case.check(out, lse)


def test_many_sequences(cuda_lib):
    """More sequences than a block has threads, most of them short, some empty."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(5)
    starts = [int(x) for x in rng.integers(-3, 40, 900)]
    starts[700], starts[899] = 300, 200
    case = Case(51, starts, [int(x) for x in rng.integers(0, 3, 900)], 2, 4, 2)
    cache, start, a = case.arguments()
    want = case.want()
    for shares in (0, 5, 300):
        out, lse = kernels.attention_tree(dev(case.q), cache, start, want_lse=True, shares=shares, **a)
        case.check(out, lse, want)
    weight = dev(case.c.weight)
    kernels.kv8_weigh(dev(case.q), lse, cache, weight, start, **a)
    assert abs(float(weight.double().sum()) - case.c.weight.astype(np.float64).sum() - (~np.isneginf(want[1])).sum()) < 1e-2


def test_no_room_for_cuts(cuda_lib):
    from tenzo_b200 import kernels
    case = Case(1, [3000, 10, 400], [4, 4, 2], 4, 20, 5)
    cache, start, a = case.arguments()
    for size in (0, 100, 5000):
        out, lse = kernels.attention_tree(dev(case.q), cache, start, want_lse=True, workspace=torch.empty(size, dtype=torch.uint8, device="cuda"), **a)
        case.check(out, lse)
    with pytest.raises(RuntimeError):
        kernels.attention_tree(dev(case.q), cache, start, shares=20, workspace=torch.empty(5000, dtype=torch.uint8, device="cuda"), **a)


def test_growing_scores(cuda_lib):
    """The largest argument moves on from tile to tile, in some rows, by much and by little; values' scales grow too."""
    from tenzo_b200 import kernels
    for step in (0.02, 0.5, 6.0):
        case = Case(7, [1300], [16], 16, 20, 5, rotated=False, masked=False)
        b, o = case.c.at(0, np.arange(1316))
        case.c.k[b, 0, :, o] = np.sign(case.q[3].reshape(5, 4, 128)[:, 0]).astype(np.int8) * 20      # along one query of each kv head
        case.c.sk[b, 0, :, o] = (0.02 * step * (1 + np.arange(1316) // 100))[:, None]
        case.c.sv[b, 0, :, o] = (0.001 * 1.5 ** (np.arange(1316) // 90))[:, None]
        cache, start, a = case.arguments()
        out, lse = kernels.attention_tree(dev(case.q), cache, start, want_lse=True, **a)
        want_out, want_lse, bound, lse_bound, _ = case.want()
        assert (np.abs(host(out) - want_out) <= bound).all() and (np.abs(host(lse) - want_lse) <= lse_bound).all()


def test_masks_that_leave_nothing(cuda_lib):
    """Rows that see no key at all, not even their own; rows that see only others'."""
    from tenzo_b200 import kernels
    case = Case(2, [0, 0, 200], [40, 40, 40], 40, 20, 5)
    for i in range(0, 120, 3):
        case.sees[i] = set()
    case.sees[1] = {39}
    case.sees[41] = {0, 31, 32}
    cache, start, a = case.arguments()
    out, lse = kernels.attention_tree(dev(case.q), cache, start, want_lse=True, **a)
    case.check(out, lse)
    weight = torch.zeros_like(dev(case.c.weight))
    kernels.kv8_weigh(dev(case.q), lse, cache, weight, start, **a)
    assert torch.isfinite(weight).all() and abs(float(weight.double().sum()) - 20 * int((~np.isneginf(host(lse))).sum() / 20)) < 1e-3


def test_queries_that_are_not_finite(cuda_lib):
    """They spoil their own head's row and no other; nor do they pass into weights."""
    from tenzo_b200 import kernels
    case = Case(3, [300], [10], 10, 20, 5)
    good = case.want()
    case.q[2, 128 * 7 + 5], case.q[4, 128 * 19 + 127], case.q[9, 0] = np.nan, np.inf, -np.inf
    cache, start, a = case.arguments()
    out, lse = kernels.attention_tree(dev(case.q), cache, start, want_lse=True, **a)
    bad = np.zeros((10, 20), bool)
    bad[2, 7] = bad[4, 19] = bad[9, 0] = True
    assert np.array_equal(np.isnan(host(lse)), bad) and np.array_equal(np.isnan(host(out)), np.repeat(bad, 128, 1))
    fine = ~np.repeat(bad, 128, 1)
    assert (np.abs(host(out) - good[0])[fine] <= good[2][fine]).all()
    weight = torch.zeros_like(dev(case.c.weight))
    kernels.kv8_weigh(dev(case.q), lse, cache, weight, start, **a)
    assert abs(float(weight.double().sum()) - 197) < 1e-3


def test_keys_and_values_that_are_not_finite(cuda_lib):
    """A scale that is no number spoils the rows that see it, and those alone."""
    from tenzo_b200 import kernels
    case = Case(13, [200], [12], 12, 20, 5)
    (b, o), (d, e) = case.c.at(0, 205), case.c.at(0, 209)
    case.c.sk[b, 0, 1, o] = np.nan
    case.c.sv[d, 0, 3, e] = np.inf
    cache, start, a = case.arguments()
    out = host(kernels.attention_tree(dev(case.q), cache, start, **a)).reshape(12, 20, 128)
    for i in range(12):
        assert np.isfinite(out[i, 4:8]).all() == (5 not in case.sees[i]) and np.isfinite(out[i, 12:16]).all() == (9 not in case.sees[i])
        assert np.isfinite(out[i, :4]).all() and np.isfinite(out[i, 8:12]).all() and np.isfinite(out[i, 16:]).all()


def test_table_rows_and_strided_queries(cuda_lib):
    from tenzo_b200 import kernels
    case = Case(4, [70, 150, 20], [6, 6, 6], 6, 20, 5)
    cache, start, a = case.arguments()
    wide = torch.full((18, 3 + 20 * 128 + 5), float("nan"), device="cuda")
    wide[:, 3: 3 + 2560] = dev(case.q)
    order = [2, 0, 1]
    back = np.argsort(order)
    shuffled = kernels.Kv8Cache(*cache[:4], cache.block_table[torch.tensor(back, device="cuda")].contiguous())
    seq = dev(np.array(order, np.int32))
    out, lse = kernels.attention_tree(wide[:, 3: 3 + 2560], shuffled, start, seq=seq, want_lse=True, **a)
    want = case.want()
    case.check(out, lse, want)
    check_weights(case, wide[:, 3: 3 + 2560], lse, shuffled, start, a | dict(seq=seq), want)


@pytest.mark.parametrize("starts,counts,nodes", [([100, 7], [12, 9], 12), ([1500, 900], [1, 1], 1)])
def test_positions_by_default(cuda_lib, starts, counts, nodes):
    """Without rope_pos a node's position is its place."""
    from tenzo_b200 import kernels
    case = Case(nodes, starts, counts, nodes, 20, 5)
    case.pos = (np.array(starts)[:, None] + np.arange(nodes)).astype(np.int32).flatten()
    cache, start, a = case.arguments()
    del a["rope_pos"]
    q = dev(case.q)
    out, lse = kernels.attention_tree(q, cache, start, want_lse=True, **a)
    want = case.want()
    case.check(out, lse, want)
    check_weights(case, q, lse, cache, start, a, want)


def test_one_table_row_for_several_sequences(cuda_lib):
    """Drafts of one sequence that end at different tokens, and a table whose rows share blocks: attention reads what others read too."""
    from tenzo_b200 import kernels
    case = Case(17, [300, 300, 300], [6, 6, 6], 6, 20, 5)
    cache, start, a = case.arguments()
    q = dev(case.q)
    table = cache.block_table.clone()
    table[1] = table[2] = table[0]
    seq = torch.zeros(3, dtype=torch.int32, device="cuda")
    got = [kernels.attention_tree(q, kernels.Kv8Cache(*cache[:4], t), start, seq=s, want_lse=True, **a) for t, s in ((table, None), (cache.block_table, seq))]
    assert all(torch.equal(x, y) for x, y in zip(*got))
    case.c.table[1] = case.c.table[2] = case.c.table[0]
    case.check(*got[0])


def test_nothing_to_do(cuda_lib):
    from tenzo_b200 import kernels
    case = Case(19, [20], [4], 4, 20, 5)
    cache, start, a = case.arguments()
    none = {n: x[:0] if n in ("count", "mask", "rope_pos") else x for n, x in a.items()}
    out, lse = kernels.attention_tree(dev(case.q)[:0], cache, start[:0], want_lse=True, **none)
    assert out.shape == (0, 2560) and lse.shape == (0, 20)
    kernels.kv8_weigh(dev(case.q)[:0], lse, cache, dev(case.c.weight), start[:0], **none)
    with pytest.raises(RuntimeError):
        q = dev(case.q)
        kernels.attention_tree(q, cache, start, out=q, **a)


def test_out_of_range(cuda_lib):
    """Sequences and rows that are refused are left as they were, their weights too; a bad table entry leaves its block's keys out."""
    from tenzo_b200 import kernels
    case = Case(6, [100, 90, 80, 70, 60], [9, 9, 9, 9, 9], 9, 20, 5, spare=32)
    cache, start, a = case.arguments()
    a["max_len"] = 109
    start = dev(np.array([101, 90, 80, 70, 60], np.int32))                   # too long, too many nodes, no such table row, a bad position, a bad entry
    a["count"] = dev(np.array([9, 10, 9, 9, 9], np.int32))
    seq = dev(np.array([0, 1, 5, 3, 4], np.int32))
    a["rope_pos"][3 * 9 + 2], a["rope_pos"][3 * 9 + 4] = -1, len(case.cos)
    table = cache.block_table.clone()
    table[4, 2] = case.c.n_blocks
    cache = kernels.Kv8Cache(*cache[:4], table)
    out, lse = torch.full((45, 2560), 7.0, device="cuda"), torch.full((45, 20), 7.0, device="cuda")
    kernels.attention_tree(dev(case.q), cache, start, seq=seq, out=out, lse=lse, **a)
    assert kernels.kv8_take_errors() == 2
    left = list(range(27)) + [29, 31]
    assert bool((out[left] == 7).all()) and bool((lse[left] == 7).all())
    good = case.want()
    rows = [r for r in range(27, 36) if r not in left]
    assert (np.abs(host(out) - good[0])[rows] <= good[2][rows]).all()
    case.c.sk[case.c.table[4, 2], 0, :, :] = -1e30                            # as if those keys had no weight
    case.c.k[case.c.table[4, 2], 0] = 1
    x = torch.isfinite(out[36:]).all()
    assert bool(x)
    weight = dev(case.c.weight)
    kernels.kv8_weigh(dev(case.q), lse, cache, weight, start, seq=seq, **a)
    assert kernels.kv8_take_errors() == 2
    touched = np.zeros(case.c.weight.shape, bool)
    for s, n in ((3, 79), (4, 69)):
        b, o = case.c.at(s, np.arange(n))
        ok = b != case.c.table[4, 2]
        touched[b[ok], 0, :, o[ok]] = True
    got = host(weight)
    assert np.array_equal(got[~touched], case.c.weight[~touched])
    total = float((got.astype(np.float64) - case.c.weight)[touched].sum())
    assert abs(total - 20 * (7 + 9)) < 1e-2                                   # the bad entry's keys had no part in its rows' sums either


def test_equal_calls_give_equal_bits(cuda_lib):
    from tenzo_b200 import kernels
    case = Case(21, [900, 333], [64, 50], 64, 20, 5)
    cache, start, a = case.arguments()
    q, got = dev(case.q), []
    for _ in range(3):
        weight = torch.zeros_like(dev(case.c.weight))
        out, lse = kernels.attention_tree(q, cache, start, want_lse=True, **a)
        kernels.kv8_weigh(q, lse, cache, weight, start, **a)
        got.append((out, lse, weight))
    assert all(torch.equal(x, y) for g in got[1:] for x, y in zip(g, got[0]))


def test_captured_for_growing_sequences_on_two_streams(cuda_lib):
    """Two graphs of their own, replayed at the same time while the lengths grow."""
    from tenzo_b200 import kernels
    cases = [Case(31 + i, [700, 250], [12, 12], 12, 20, 5) for i in range(2)]
    sets, graphs, streams = [], [], [torch.cuda.Stream() for _ in cases]
    for case, stream in zip(cases, streams):
        cache, start, a = case.arguments()
        q = dev(case.q)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out, lse = kernels.attention_tree(q, cache, start, want_lse=True, use_pdl=True, **a)
        graphs.append(graph)
        sets.append((start, out, lse, q, cache, a))                           # (a graph does not keep what it reads)
    for grown in ([1, 200], [300, 250], [700, 3]):
        for case, (start, *_) in zip(cases, sets):
            case.starts = grown
            start.copy_(dev(np.array(grown, np.int32)))
            for s, n in enumerate(grown):                                     # (the codes there are of the same kind; a tree's rows lie behind the new length)
                assert n + 12 <= [712, 262][s]
        torch.cuda.synchronize()
        for _ in range(5):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for case, (_, out, lse, *_) in zip(cases, sets):
            case.check(out, lse)


def test_places_beyond_32_bits_of_bytes(cuda_lib):
    """A pool of more than 2^31 bytes, the sequence in its last blocks."""
    from tenzo_b200 import kernels
    case = Case(41, [90], [4], 4, 4, 1, slots=16)
    blocks = (1 << 20) + 4 * 1024                                             # 2.15 GB of keys
    far = np.arange(blocks - case.c.table.size, blocks).astype(np.int32).reshape(case.c.table.shape)
    cache, start, a = case.arguments()
    big = [torch.zeros(blocks, 1, 1, 16, 128, dtype=torch.int8, device="cuda") for _ in range(2)] + [torch.zeros(blocks, 1, 1, 16, device="cuda") for _ in range(2)]
    for x, y in zip(big, cache[:4]):
        x[torch.from_numpy(far.astype(np.int64)).cuda()] = y[cache.block_table.long()]
    out, lse = kernels.attention_tree(dev(case.q), kernels.Kv8Cache(*big, dev(far)), start, want_lse=True, **a)
    case.check(out, lse)
