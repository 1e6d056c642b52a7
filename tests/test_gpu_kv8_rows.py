"""Rows of the INT8 caches on the GPU: stored rows, accepted nodes and evictions leave the pools as the definitions do, bit for bit, and no other byte changes."""
import numpy as np
import pytest
import torch
import kv8_reference as ref
from gpu_helpers import Guarded, dev, host

pytestmark = pytest.mark.gpu


class OnGpu:
    """The pools of ref.Caches between guards."""

    def __init__(self, c):
        from tenzo_b200 import kernels
        self.guard = Guarded()
        kinds = dict(k=torch.int8, v=torch.int8, sk=torch.float32, sv=torch.float32, weight=torch.float32, position=torch.int32)
        for n, kind in kinds.items():
            x = getattr(c, n)
            setattr(self, n, self.guard.empty(x.shape, kind, dev(x)))
        self.table = dev(c.table)
        self.cache = kernels.Kv8Cache(self.k, self.v, self.sk, self.sv, self.table)

    def check(self, c):
        """The pools that differ from c's, and the guards."""
        torch.cuda.synchronize()
        for raw, n in self.guard.raws:
            assert bool((raw[:Guarded.PAD] == 0xA5).all()) and bool((raw[Guarded.PAD + n:] == 0xA5).all())
        assert [n for n in c.POOLS if host(getattr(self, n)).tobytes() != getattr(c, n).tobytes()] == []


@pytest.mark.parametrize("n_seq,tokens,start,n_kv,layers,layer,slots,rotated,padded", [
    (1, 1, 0, 5, 1, 0, 16, True, False),
    (3, 1, 15, 1, 2, 1, 16, True, False),
    (2, 37, 11, 5, 3, 1, 16, True, True),
    (5, 16, 16, 8, 1, 0, 48, False, False),
    (1, 133, 0, 2, 1, 0, 144, True, False),
    (64, 1, 200, 5, 2, 0, 16, True, True),
])
def test_append(cuda_lib, n_seq, tokens, start, n_kv, layers, layer, slots, rotated, padded):
    from tenzo_b200 import kernels
    rng = np.random.default_rng(n_seq * 1000 + tokens)
    c = ref.Caches(rng, n_seq, (start + tokens + slots - 1) // slots, layers, n_kv, slots)
    seq, place = np.repeat(np.arange(n_seq), tokens).astype(np.int32), np.tile(start + np.arange(tokens), n_seq).astype(np.int32)
    order = rng.permutation(len(place))
    seq, place = seq[order], place[order]
    pos = (rng.integers(0, 50, len(place)) + place).astype(np.int32)
    if padded:
        place[rng.random(len(place)) < 0.3] = -1
    k, v = (rng.standard_normal((len(place), n_kv * 128)).astype(np.float32) * 3 for _ in range(2))
    k[0] = 0
    v[-1, :128] = np.float32(2.5) / 127 * np.arange(-64, 64)                # halves
    cos, sin = ref.rope(start + tokens + 50)
    g = OnGpu(c)
    tables = dict(rope_cos=dev(cos), rope_sin=dev(sin), rope_pos=dev(pos)) if rotated else {}
    kernels.kv8_append(dev(k), dev(v), g.cache, dev(place), layer=layer, seq=dev(seq), weight=g.weight, position=g.position, **tables)
    for i in range(len(place)):
        if place[i] < 0:
            continue
        b, o = c.at(seq[i], place[i])
        key = k[i].reshape(n_kv, 128)
        c.k[b, layer, :, o], c.sk[b, layer, :, o] = ref.quantise(ref.rotate32(key, cos[pos[i]], sin[pos[i]]) if rotated else key)
        c.v[b, layer, :, o], c.sv[b, layer, :, o] = ref.quantise(v[i].reshape(n_kv, 128))
        c.weight[b, layer, :, o], c.position[b, layer, :, o] = 0, pos[i] if rotated else place[i]
    g.check(c)
    assert kernels.kv8_take_errors() == 0


def test_append_stores_what_the_decode_step_does(cuda_lib):
    """attention_int8 with append divides by 127 where this multiplies by 1/127: scales that differ by less than two steps, and codes by one next to a border."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(3)
    n, n_kv, max_seq = 6, 5, 64
    q, k, v = (dev(rng.standard_normal((n, h * 128)).astype(np.float32)) for h in (20, n_kv, n_kv))
    pos = dev(np.array([0, 3, 15, 16, 40, 63], np.int32))
    cos, sin = (dev(x) for x in ref.rope(max_seq))
    caches = [[torch.zeros(n, 2, n_kv, max_seq, 128, dtype=torch.int8, device="cuda") for _ in range(2)] + [torch.zeros(n, 2, n_kv, max_seq, device="cuda") for _ in range(2)] for _ in range(2)]
    kernels.attention_int8(q, k, v, *caches[0], pos, layer=1, n_q=20, n_kv=n_kv, max_seq=max_seq, rope_cos=cos, rope_sin=sin)
    kernels.kv8_append(k, v, kernels.Kv8Cache(*caches[1], torch.arange(n, dtype=torch.int32, device="cuda")[:, None]), pos, layer=1, rope_cos=cos, rope_sin=sin)
    for a, b in zip(caches[0][2:], caches[1][2:]):
        assert bool(((a - b).abs() <= 2 ** -22 * a).all()) and bool(((a > 0) == (b > 0)).all()) and int((a > 0).sum()) == n * n_kv
    for a, b in zip(caches[0][:2], caches[1][:2]):
        assert int((a.int() - b.int()).abs().max()) <= 1 and int((a != b).sum()) <= 2          # (a code in some millions)


def test_append_strided_rows(cuda_lib):
    """Rows that are slices of a wider buffer, aligned to four bytes only."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(8)
    c = ref.Caches(rng, 1, 3, 1, 2, 16)
    wide = dev(rng.standard_normal((20, 1 + 2 * 256 + 3)).astype(np.float32))
    k, v = wide[:, 1:257], wide[:, 257:513]
    g, h = OnGpu(c), OnGpu(c)
    place, seq = torch.arange(5, 25, dtype=torch.int32, device="cuda"), torch.zeros(20, dtype=torch.int32, device="cuda")
    kernels.kv8_append(k, v, g.cache, place, layer=0, seq=seq)
    kernels.kv8_append(k.contiguous(), v.contiguous(), h.cache, place, layer=0, seq=seq)
    assert all(torch.equal(getattr(g, n).view(torch.uint8), getattr(h, n).view(torch.uint8)) for n in c.POOLS)


def test_append_out_of_range(cuda_lib):
    from tenzo_b200 import kernels
    rng = np.random.default_rng(4)
    c = ref.Caches(rng, 2, 3, 1, 2, 16)
    c.table[1, 1] = c.n_blocks
    g = OnGpu(c)
    place = dev(np.array([48, 3, 3, 17, 5, 5], np.int32))
    seq, pos = dev(np.array([0, 2, -1, 1, 0, 0], np.int32)), dev(np.array([1, 1, 1, 1, 30, -1], np.int32))
    cos, sin = (dev(x) for x in ref.rope(30))
    x = torch.ones(6, 256, device="cuda")
    kernels.kv8_append(x, x, g.cache, place, layer=0, seq=seq, rope_pos=pos, rope_cos=cos, rope_sin=sin, weight=g.weight, position=g.position)
    g.check(c)
    assert kernels.kv8_take_errors() == 2 and kernels.kv8_take_errors() == 0


def evict_case(rng, lengths, layers, n_kv, slots, levels=None):
    n = max(lengths)
    c = ref.Caches(rng, len(lengths), (n + slots - 1) // slots, layers, n_kv, slots)
    for s, m in enumerate(lengths):
        c.fill(rng, s, range(m))
    if levels:                                       # weights of few values: ties
        c.weight[:] = rng.integers(0, levels, c.weight.shape).astype(np.float32) / 4
    return c


@pytest.mark.parametrize("lengths,keep,recent,layers,n_kv,slots,levels", [
    ([1], 1, 0, 1, 1, 16, None),
    ([2], 1, 1, 1, 1, 16, None),
    ([40, 39, 100, 16], 39, 5, 2, 3, 16, None),
    ([700, 513], 512, 64, 2, 2, 16, 5),
    ([700, 300], 17, 0, 1, 3, 704, 1),
    ([33, 65, 64], 32, 40, 1, 2, 80, 2),
    ([2177], 2048, 256, 1, 5, 16, None),
    ([5000, 1], 4999, 3, 1, 1, 16, 3),
    ([33 + 37 * s % 90 for s in range(40)], 40, 6, 5, 3, 16, 40),             # (more CTAs than the GPU holds of the larger ones)
    ([700 + 97 * s % 900 for s in range(40)], 690, 64, 5, 3, 16, None),
])
def test_evict(cuda_lib, lengths, keep, recent, layers, n_kv, slots, levels):
    from tenzo_b200 import kernels
    rng = np.random.default_rng(sum(lengths) + keep)
    c = evict_case(rng, lengths, layers, n_kv, slots, levels)
    for s, n in enumerate(lengths):                  # newest tokens anywhere
        b, o = c.at(s, np.arange(n))
        for layer in range(layers):
            for h in range(n_kv):
                c.position[b, layer, h, o] = rng.permutation(n) + 10 * s
    start = np.array([n - recent + 10 * s for s, n in enumerate(lengths)], np.int32)
    g = OnGpu(c)
    got = kernels.kv8_evict(g.cache, g.weight, g.position, dev(np.array(lengths, np.int32)), keep=keep, protect_from=dev(start) if recent else None, max_len=max(lengths))
    want = [ref.evict(c, s, n, keep, start[s] if recent else None) for s, n in enumerate(lengths)]
    g.check(c)
    assert host(got).tolist() == want and kernels.kv8_take_errors() == 0


def test_evict_special_weights(cuda_lib):
    """Infinities, zeros of both signs, subnormals, negative ones and NaN."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(9)
    special = np.array([np.inf, -np.inf, 0.0, -0.0, 1e-42, -1e-42, np.nan, 3.0, -3.0, 65504.0], np.float32)
    for keep in (1, 7, 50, 99):
        c = evict_case(rng, [100], 1, 3, 16)
        c.weight[:] = rng.choice(special, c.weight.shape)
        g = OnGpu(c)
        kernels.kv8_evict(g.cache, g.weight, g.position, dev(np.array([100], np.int32)), keep=keep)
        ref.evict(c, 0, 100, keep, None)
        g.check(c)


@pytest.mark.parametrize("n,keep", [(60000, 59000), (60000, 20000), (49153, 30000), (49152, 49151)])
def test_evict_long(cuda_lib, n, keep):
    """Caches of more tokens than shared memory has room for, and lists of more than it has room for at a time."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(n + keep)
    c = ref.Caches(rng, 1, (n + 15) // 16, 1, 1, 16)
    c.sk[:], c.sv[:] = rng.random(c.sk.shape), rng.random(c.sv.shape)
    g = OnGpu(c)
    kernels.kv8_evict(g.cache, g.weight, g.position, dev(np.array([n], np.int32)), keep=keep, protect_from=dev(np.array([1 << 19], np.int32)), max_len=n)
    ref.evict(c, 0, n, keep, 1 << 19)
    g.check(c)


def test_evict_rows_of_the_table_and_out_of_range(cuda_lib):
    from tenzo_b200 import kernels
    rng = np.random.default_rng(11)
    c = evict_case(rng, [64, 64, 64, 64], 2, 2, 16)
    c.table[2, 3] = -1
    g = OnGpu(c)
    length, seq = [60, 50, -1, 65, 64, 30], [3, 0, 1, 1, 2, 4]      # the third and fourth have no such length, the fifth a bad entry, the sixth no such row
    got = kernels.kv8_evict(g.cache, g.weight, g.position, dev(np.array(length, np.int32)), keep=20, seq=dev(np.array(seq, np.int32)), max_len=64)
    ref.evict(c, 3, 60, 20, None)
    ref.evict(c, 0, 50, 20, None)
    g.check(c)
    assert host(got).tolist() == [20, 20, -1, 65, 64, 30] and kernels.kv8_take_errors() == 2


@pytest.mark.parametrize("nodes,counts,starts,layers,n_kv,slots", [
    (1, [1], [0], 1, 1, 16),
    (2, [2, 1, 2], [15, 16, 0], 2, 3, 16),
    (24, [24], [219], 30, 5, 16),
    (33, [33, 20, 0, 7], [100, 31, 5, 0], 3, 2, 16),
    (256, [256, 255], [9, 300], 2, 2, 16),
    (64, [64, 64, 50], [0, 7, 77], 2, 4, 144),
])
def test_accept(cuda_lib, nodes, counts, starts, layers, n_kv, slots):
    from tenzo_b200 import kernels
    rng = np.random.default_rng(nodes + sum(starts))
    n_seq = len(counts)
    c = ref.Caches(rng, n_seq, (max(starts) + nodes + slots - 1) // slots, layers, n_kv, slots)
    parent = np.array([[max(-1, i - 1 - int(rng.integers(0, 4))) for i in range(nodes)] for _ in range(n_seq)], np.int32)
    parent[:, 1:] = np.maximum(parent[:, 1:], 0)
    token = rng.integers(0, 3, (n_seq, nodes)).astype(np.int32)              # few tokens: long paths, and children of equal tokens
    chosen = rng.integers(0, 3, (n_seq, nodes)).astype(np.int32)
    for s in range(n_seq):                                                     # one line of each tree is agreed with for a while
        i = counts[s] - 1
        while i > 0 and rng.random() < 0.97:
            chosen[s, parent[s, i]] = token[s, i]
            i = parent[s, i]
    g = OnGpu(c)
    accepted, following, path = kernels.kv8_accept(g.cache, dev(token), dev(parent), dev(chosen), dev(np.array(starts, np.int32)), count=dev(np.array(counts, np.int32)),
                                                   weight=g.weight, position=g.position)
    for s in range(n_seq):
        want, then = ref.accept(c, s, starts[s], token[s, : counts[s]], parent[s], chosen[s])
        assert host(path[s]).tolist() == want + [-1] * (nodes - len(want)) and int(accepted[s]) == len(want) and int(following[s]) == then
    g.check(c)
    assert kernels.kv8_take_errors() == 0


def test_accept_a_line_with_gaps(cuda_lib):
    """The longest way that rows can move: every second node, so that old and new places overlap."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(5)
    nodes = 256
    c = ref.Caches(rng, 1, 17, 3, 4, 16)
    parent = np.array([[-1, 0] + [(i - 2) // 2 * 2 for i in range(2, nodes)]], np.int32)
    token, chosen = np.arange(nodes, dtype=np.int32)[None], np.array([[i + 2 for i in range(nodes)]], np.int32)
    g = OnGpu(c)
    _, _, path = kernels.kv8_accept(g.cache, dev(token), dev(parent), dev(chosen), dev(np.array([3], np.int32)))
    want, _ = ref.accept(c, 0, 3, token[0], parent[0], chosen[0])
    assert len(want) == 128 and host(path[0])[:128].tolist() == want
    c.weight, c.position = host(g.weight), host(g.position)                    # were not given
    g.check(c)


def test_accept_padding_bad_parents_and_out_of_range(cuda_lib):
    from tenzo_b200 import kernels
    rng = np.random.default_rng(6)
    c = ref.Caches(rng, 6, 2, 1, 2, 16)
    c.table[5, 1] = 1 << 20
    g = OnGpu(c)
    parent = np.tile(np.array([-1, 0, 5, 1, -7], np.int32), (7, 1))           # a parent behind its child, and one that is none: never reached
    token, chosen = np.tile(np.array([4, 6, 6, 9, 6], np.int32), (7, 1)), np.tile(np.array([6, 9, 9, 9, 1], np.int32), (7, 1))
    parent[5], token[5], chosen[5] = [-1, 0, 0, 2, 3], [0, 1, 2, 3, 4], [2, 1, 3, 4, 8]
    start, count, seq = np.array([3, -2, 3, 28, 3, 13, 3], np.int32), np.array([5, 5, 0, 5, 6, 5, 5], np.int32), np.array([0, 1, 2, 3, 4, 5, 6], np.int32)
    accepted, following, path = kernels.kv8_accept(g.cache, dev(token), dev(parent), dev(chosen), dev(start), count=dev(count), seq=dev(seq), weight=g.weight, position=g.position)
    assert host(accepted).tolist() == [3, 0, 0, 0, 0, 4, 0] and host(following).tolist() == [9, -1, -1, -1, -1, 8, -1]
    assert host(path[0]).tolist() == [0, 1, 3, -1, -1] and host(path[5]).tolist() == [0, 2, 3, 4, -1] and bool((path[[1, 2, 3, 4, 6]] == -1).all())
    ref.accept(c, 0, 3, token[0], parent[0], chosen[0])
    (a, b), (d, e) = c.at(5, 15), c.at(5, 14)                                 # of the sixth sequence one row has both its places
    assert kernels.kv8_take_errors() == 2
    for n in c.POOLS:
        getattr(c, n)[d, :, :, e] = getattr(c, n)[a, :, :, b]
    g.check(c)


@pytest.mark.parametrize("what", ["append", "evict", "accept"])
def test_captured_and_on_another_stream(cuda_lib, what):
    """A call captured once, with new inputs before each replay, on a stream of its own."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(12)
    c = evict_case(rng, [60, 50], 2, 2, 16)
    g = OnGpu(c)
    ints = lambda *x: dev(np.array(x, np.int32))                               # noqa: E731
    length, place, seq = ints(60, 50), ints(3, 47), ints(0, 1)
    rows = torch.zeros(2, 256, device="cuda")
    token, parent, chosen, start = ints(1, 2, 3, 4).expand(2, 4).contiguous(), ints(-1, 0, 0, 2).expand(2, 4).contiguous(), ints(3, 0, 4, 9).expand(2, 4).contiguous(), ints(7, 30)

    def call():
        if what == "append":
            kernels.kv8_append(rows, rows, g.cache, place, layer=1, seq=seq, weight=g.weight, position=g.position, use_pdl=True)
        elif what == "evict":
            kernels.kv8_evict(g.cache, g.weight, g.position, length, keep=40, max_len=60, use_pdl=True)
        else:
            kernels.kv8_accept(g.cache, token, parent, chosen, start, weight=g.weight, position=g.position, use_pdl=True)

    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        call()
    for turn in range(3):
        x = rng.standard_normal((2, 256)).astype(np.float32)
        rows.copy_(dev(x))
        start.copy_(ints(7 + turn, 30 - turn))
        length.copy_(ints(60 - turn, 50 + turn))
        graph.replay()
        for s in range(2):
            if what == "append":
                b, o = c.at(s, int(place[s]))
                for code, scale in ((c.k, c.sk), (c.v, c.sv)):
                    code[b, 1, :, o], scale[b, 1, :, o] = ref.quantise(x[s].reshape(2, 128))
                c.weight[b, 1, :, o], c.position[b, 1, :, o] = 0, int(place[s])
            elif what == "evict":
                ref.evict(c, s, int(length[s]), 40, None)
            else:
                ref.accept(c, s, int(start[s]), host(token[s]), host(parent[s]), host(chosen[s]))
        g.check(c)
    assert kernels.kv8_take_errors() == 0
