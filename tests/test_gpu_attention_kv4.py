"""Attention over the 4-bit paged cache against the formula in 64 bits (kv4_reference.attention derives the bound)."""
import numpy as np
import pytest
import torch
import kv4_reference as ref
from gpu_helpers import Guarded, dev, host

pytestmark = pytest.mark.gpu


def setup(rng, lens, n_kv, columns, layers=1, spread=1.0, garbage=True):
    """A pool whose slots behind a sequence's last key, and whose other blocks, hold anything (NaN parameters among it)."""
    n_seq = len(lens)
    blocks = n_seq * columns + 2
    table = rng.permutation(blocks)[: n_seq * columns].astype(np.int32).reshape(n_seq, columns)
    pool = rng.integers(0, 256, (blocks, layers, n_kv, 2, 16, 80), dtype=np.uint8) if garbage else np.zeros((blocks, layers, n_kv, 2, 16, 80), np.uint8)
    if garbage:
        pool[..., 64:] = np.array([0x7E00, 0x7C00], np.uint16).view(np.uint8).tolist() * 4           # NaN, infinity
    good = ref.random_pool(rng, blocks, layers, n_kv, spread)
    for s, n in enumerate(lens):
        for c in range((n + 15) // 16):
            m = min(16, n - 16 * c)
            pool[table[s, c], :, :, :, :m] = good[table[s, c], :, :, :, :m]
    return table, pool


def check(out, q, pool, table, layer, pos, seq, cos=None, sin=None):
    n_q = q.shape[1] // 128
    for i, (p, s) in enumerate(zip(pos, seq)):
        k, v = ref.cached(pool, layer, table[s], max(0, p + 1))
        turn = (cos[p], sin[p]) if cos is not None and p >= 0 else (None, None)
        want, bound = ref.attention(q[i].reshape(n_q, 128), k, v, *turn)
        err = abs(out[i].reshape(n_q, 128).astype(np.float64) - want)
        assert (err <= bound).all(), (i, p, float((err / bound).max()))
        if p >= 0:                                               # and on the whole, to the type's own accuracy
            rel = np.linalg.norm(out[i].reshape(n_q, 128) - want) / np.linalg.norm(want)
            assert rel <= 2e-6, (i, p, rel)


LENS = [1, 2, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 0, 200, 255, 256, 257, 300]


@pytest.mark.parametrize("n_q,n_kv", [(20, 5), (4, 4), (2, 1), (3, 1), (6, 1), (7, 1), (8, 1), (16, 2), (9, 1), (16, 1), (20, 1), (33, 1)])
@pytest.mark.parametrize("split", [0, 128])
def test_lengths_and_heads(cuda_lib, n_q, n_kv, split):
    from tenzo_b200 import kernels
    rng = np.random.default_rng(n_q * 100 + n_kv)
    table, pool = setup(rng, LENS, n_kv, 20)
    q = rng.standard_normal((len(LENS), n_q * 128)).astype(np.float32) * 2
    pos = np.array(LENS, np.int32) - 1
    cos, sin = ref.rope(320)
    g = Guarded()
    out = g.empty((len(LENS), n_q * 128), torch.float32)
    ws = g.empty((kernels.attention_kv4_workspace_bytes(len(LENS), n_q, n_kv, 320),), torch.uint8)
    kernels.attention_kv4(dev(q), dev(pool), dev(pos), layer=0, n_q=n_q, block_table=dev(table), rope_cos=dev(cos), rope_sin=dev(sin), out=out, split_keys=split,
                          workspace=ws)
    check(host(out), q, pool, table, 0, pos, range(len(LENS)), cos, sin)
    g.check()
    assert kernels.kv4_take_errors() == 0


@pytest.mark.parametrize("n_q,n_kv,lens", [(20, 5, [5000, 4097, 1]), (16, 2, [9001]), (12, 4, [1234, 3000, 2048, 77]), (32, 8, [16000])])
def test_long_contexts(cuda_lib, n_q, n_kv, lens):
    """Every way of splitting gives the result: chosen, forced, and with a workspace that allows some splits or none."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(sum(lens))
    most = max(lens)
    table, pool = setup(rng, lens, n_kv, (most + 15) // 16, layers=2)
    q = rng.standard_normal((len(lens), n_q * 128)).astype(np.float32)
    pos = np.array(lens, np.int32) - 1
    dq, dp, dpos, dt = dev(q), dev(pool), dev(pos), dev(table)
    full = kernels.attention_kv4_workspace_bytes(len(lens), n_q, n_kv, most)
    for split, room in ((0, full), (256, full), (1000, full), (0, full // 3), (0, 0), (most, 0)):
        ws = torch.empty(max(room, 16), dtype=torch.uint8, device="cuda")[:room]
        out = kernels.attention_kv4(dq, dp, dpos, layer=1, n_q=n_q, block_table=dt, max_len=most, split_keys=split, workspace=ws)
        check(host(out), q, pool, table, 1, pos, range(len(lens)))
    assert kernels.kv4_take_errors() == 0


@pytest.mark.parametrize("scale_q,spread", [(1e-6, 1.0), (1.0, 1e-3), (1.0, 300.0), (30.0, 1.0), (0.0, 1.0), (1e4, 1e-4)])
def test_magnitudes(cuda_lib, scale_q, spread):
    """Queries and values far from 1: nothing overflows or fades in the 16-bit parts of the products."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(3)
    lens = [33, 700]
    table, pool = setup(rng, lens, 2, 44, spread=spread)
    keys = ref.random_pool(rng, len(pool), 1, 2, 1.0)
    pool[:, :, :, 0] = keys[:, :, :, 0]                                   # keys of ordinary size, values of `spread`
    q = rng.standard_normal((2, 8 * 128)).astype(np.float32) * np.float32(scale_q)
    pos = np.array(lens, np.int32) - 1
    out = kernels.attention_kv4(dev(q), dev(pool), dev(pos), layer=0, n_q=8, block_table=dev(table))
    for i, p in enumerate(pos):
        k, v = ref.cached(pool, 0, table[i], p + 1)
        want, bound = ref.attention(q[i].reshape(8, 128), k, v)
        err = abs(host(out)[i].reshape(8, 128).astype(np.float64) - want)
        assert (err <= bound).all(), float((err / bound).max())


def test_values_that_grow_along_the_sequence(cuda_lib):
    """The scale of the values rises by a factor of a million from the first key to the last, and falls in the second sequence."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(8)
    n = 640
    x = rng.standard_normal((2, n, 128)).astype(np.float32)
    grow = np.exp(np.linspace(-7, 7, n)).astype(np.float32)[:, None]
    rows_v = np.stack([ref.quantise(x[0] * grow), ref.quantise(x[1] * grow[::-1])])
    rows_k = ref.quantise(rng.standard_normal((2, n, 128)).astype(np.float32))
    pool = np.stack([rows_k, rows_v], 2).reshape(2, n // 16, 16, 2, 80).transpose(0, 1, 3, 2, 4).reshape(2 * n // 16, 1, 1, 2, 16, 80).copy()
    table = np.arange(2 * n // 16, dtype=np.int32).reshape(2, -1)
    q = rng.standard_normal((2, 4 * 128)).astype(np.float32) * 3
    pos = np.full(2, n - 1, np.int32)
    for split in (0, 128, 640):
        out = kernels.attention_kv4(dev(q), dev(pool), dev(pos), layer=0, n_q=4, block_table=dev(table), split_keys=split)
        check(host(out), q, pool, table, 0, pos, range(2))


def test_one_key_far_above_the_others(cuda_lib):
    """A score far above all others, at the first key, at the last, and growing scores (the running maximum moves at every step)."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(4)
    n = 333
    base = rng.standard_normal(128).astype(np.float32)
    x = rng.standard_normal((3, n, 128)).astype(np.float32)
    x[0, 0] = base * 6
    x[1, n - 1] = base * 6
    x[2] = base * np.linspace(-5, 5, n)[:, None].astype(np.float32) + 0.1 * x[2]
    columns = (n + 15) // 16
    rows = np.zeros((3, columns * 16, 2, 80), np.uint8)
    rows[:, :n, 0] = ref.quantise(x)
    rows[:, :n, 1] = ref.quantise(rng.standard_normal((3, n, 128)).astype(np.float32))
    pool = rows.reshape(3 * columns, 16, 2, 80).transpose(0, 2, 1, 3).reshape(3 * columns, 1, 1, 2, 16, 80).copy()
    table = np.arange(3 * columns, dtype=np.int32).reshape(3, -1)
    q = np.tile(base, (3, 2)).astype(np.float32) * np.float32(0.3)
    pos = np.full(3, n - 1, np.int32)
    out = kernels.attention_kv4(dev(q), dev(pool), dev(pos), layer=0, n_q=2, block_table=dev(table))
    check(host(out), q, pool, table, 0, pos, range(3))


def test_rows_of_one_sequence_and_shared_blocks(cuda_lib):
    """A draft's rows, each at its own position, from strided queries; tables that share blocks, as beams do; padding rows."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(12)
    table, pool = setup(rng, [100, 100], 2, 7)
    table[1, :5] = table[0, :5]
    seq = np.array([0, 0, 0, 1, 1, 1, 0, 1], np.int32)
    pos = np.array([95, 96, 97, 40, 98, 99, -1, -5], np.int32)
    wide = rng.standard_normal((8, 12 * 128)).astype(np.float32)
    d = dev(wide)
    cos, sin = ref.rope(112)
    out = kernels.attention_kv4(d[:, 128: 9 * 128], dev(pool), dev(pos), layer=0, n_q=8, block_table=dev(table), seq=dev(seq), rope_cos=dev(cos), rope_sin=dev(sin))
    check(host(out), wide[:, 128: 9 * 128], pool, table, 0, pos, seq, cos, sin)
    assert bool((out[6:] == 0).all())


def test_indices_out_of_range(cuda_lib):
    """A position past max_len or a sequence that is not there: the row stays as it was. A table entry out of range: its keys are left out."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(2)
    lens = [60, 60, 60, 60]
    table, pool = setup(rng, lens, 2, 4)
    broken = table.copy()
    broken[1, 2], broken[3, 0] = len(pool), -3
    seq = np.array([0, 1, 2, 3, 7, -1], np.int32)
    pos = np.array([59, 59, 64, 59, 3, 3], np.int32)
    q = rng.standard_normal((6, 4 * 128)).astype(np.float32)
    for split in (0, 128):
        out = torch.full((6, 4 * 128), 5.0, device="cuda")
        kernels.attention_kv4(dev(q), dev(pool), dev(pos), layer=0, n_q=4, block_table=dev(broken), seq=dev(seq), out=out, max_len=64, split_keys=split)
        assert kernels.kv4_take_errors() == 2 and kernels.kv4_take_errors() == 0
        got = host(out)
        check(got[:1], q[:1], pool, table, 0, pos[:1], seq[:1])
        assert (got[[2, 4, 5]] == 5.0).all()
        for i, gone in ((1, 2), (3, 0)):
            k, v = ref.cached(pool, 0, table[i], 60)
            keep = np.r_[0: 16 * gone, 16 * gone + 16: 60]
            want, bound = ref.attention(q[i].reshape(4, 128), k[:, keep], v[:, keep])
            assert (abs(got[i].reshape(4, 128) - want) <= bound).all()
    only_bad = np.full((1, 4), -1, np.int32)
    out = kernels.attention_kv4(dev(q[:1]), dev(pool), dev(pos[:1]), layer=0, n_q=4, block_table=dev(only_bad))
    assert kernels.kv4_take_errors() == 2 and bool((out == 0).all())


def test_two_graphs_on_one_workspace_and_a_side_stream(cuda_lib):
    from tenzo_b200 import kernels
    rng = np.random.default_rng(21)
    table, pool = setup(rng, [700, 650], 2, 44)
    q = [rng.standard_normal((2, 4 * 128)).astype(np.float32) for _ in range(2)]
    pos = np.array([699, 649], np.int32)
    dq, dp, dpos, dt = [dev(x) for x in q], dev(pool), dev(pos), dev(table)
    ws = torch.empty(kernels.attention_kv4_workspace_bytes(2, 4, 2, 704), dtype=torch.uint8, device="cuda")
    graphs, outs = [], [torch.zeros(2, 4 * 128, device="cuda") for _ in range(2)]
    side = torch.cuda.Stream()
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            for _ in range(2):
                kernels.attention_kv4(dq[i], dp, dpos, layer=0, n_q=4, block_table=dt, out=outs[i], workspace=ws, split_keys=128, use_pdl=True)
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for i in range(2):
        check(host(outs[i]), q[i], pool, table, 0, pos, range(2))
        assert torch.equal(outs[i], kernels.attention_kv4(dq[i], dp, dpos, layer=0, n_q=4, block_table=dt, split_keys=128))
    assert kernels.kv4_take_errors() == 0


@pytest.mark.parametrize("n_q,n_kv", [(4, 2), (8, 1), (12, 1)])
def test_a_prompts_rows(cuda_lib, n_q, n_kv):
    """Every position of one sequence as a row of its own, in any order."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(n_q)
    n = 700
    table, pool = setup(rng, [n], n_kv, 44)
    pos = rng.permutation(n).astype(np.int32)
    q = rng.standard_normal((n, n_q * 128)).astype(np.float32)
    cos, sin = ref.rope(n)
    out = host(kernels.attention_kv4(dev(q), dev(pool), dev(pos), layer=0, n_q=n_q, block_table=dev(table), seq=torch.zeros(n, dtype=torch.int32, device="cuda"),
                                     rope_cos=dev(cos), rope_sin=dev(sin)))
    some = rng.choice(n, 60, replace=False)
    check(out[some], q[some], pool, table, 0, pos[some], np.zeros(60, int), cos, sin)


@pytest.mark.parametrize("n_q,n_kv,lens,split", [(4, 1, [90, 70], 0), (12, 2, [3000, 2500], 0), (8, 1, [900, 1000], 0), (8, 2, [700, 600], 128)])
def test_a_query_that_is_not_finite(cuda_lib, n_q, n_kv, lens, split):
    """NaN or infinity in one head of one row: NaN there, and the other heads' bits as before."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(n_q + split)
    table, pool = setup(rng, lens, n_kv, (max(lens) + 15) // 16)
    q = rng.standard_normal((2, n_q * 128)).astype(np.float32)
    dp, dpos, dt = dev(pool), dev(np.array(lens, np.int32) - 1), dev(table)
    call = lambda x: host(kernels.attention_kv4(dev(x), dp, dpos, layer=0, n_q=n_q, block_table=dt, split_keys=split)).reshape(2, n_q, 128)
    want = call(q)
    for bad in (np.nan, np.inf, -np.inf):
        x = q.copy()
        x[1, 2 * 128 + 17] = bad
        got = call(x)
        assert np.isnan(got[1, 2]).all()
        got[1, 2] = want[1, 2]
        assert np.array_equal(got, want)


@pytest.mark.parametrize("n_q,n_kv,lens", [(20, 5, [4000]), (40, 5, [6000, 5000]), (16, 1, [3000] * 9), (8, 2, [1500] * 40)])
def test_room_for_the_chosen_splits_is_enough(cuda_lib, n_q, n_kv, lens):
    """The workspace that a call takes by itself gives the same splits, and bits, as one with room for any."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(n_q)
    table, pool = setup(rng, lens, n_kv, (max(lens) + 15) // 16, garbage=False)
    q, dp, dpos, dt = dev(rng.standard_normal((len(lens), n_q * 128)).astype(np.float32)), dev(pool), dev(np.array(lens, np.int32) - 1), dev(table)
    ws = torch.empty(kernels.attention_kv4_workspace_bytes(len(lens), n_q, n_kv, max(lens)), dtype=torch.uint8, device="cuda")
    call = lambda **kw: kernels.attention_kv4(q, dp, dpos, layer=0, n_q=n_q, block_table=dt, max_len=max(lens), **kw)
    assert torch.equal(call(), call(workspace=ws))
    assert kernels.kv4_take_errors() == 0


@pytest.mark.parametrize("n_q,n_kv", [(5, 5), (8, 4), (9, 3), (20, 5), (2, 2)])
@pytest.mark.parametrize("split", [0, 128])
def test_rows_that_share_a_sequence(cuda_lib, n_q, n_kv, split):
    """Many rows, in runs of one to twenty of the same sequence, at any positions; padding, and indices out of range, between them."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(n_q * 10 + n_kv)
    lens = [int(n) for n in rng.integers(1, 600, 40)] + [1, 16, 33]
    table, pool = setup(rng, lens, n_kv, 38, layers=2)
    seq = np.concatenate([np.full(rng.integers(1, 21) if rng.random() < 0.5 else 1, s) for s in rng.permutation(len(lens))]).astype(np.int32)
    pos = np.array([rng.integers(max(0, lens[s] - 8), lens[s]) if rng.random() < 0.7 else rng.integers(0, lens[s]) for s in seq], np.int32)
    pos[rng.random(len(pos)) < 0.1] = -1
    refused = rng.choice(len(pos), 8, replace=False)
    q = rng.standard_normal((len(seq), n_q * 128)).astype(np.float32) * 2
    cos, sin = ref.rope(608)
    g = Guarded()
    out = g.empty((len(seq), n_q * 128), torch.float32)
    for bad in (False, True):
        if bad:
            pos[refused[:4]], seq[refused[4:]] = [608, 609, 1 << 30, 700], [-1, len(lens), 1 << 30, -5]
        out.fill_(7.0)
        kernels.attention_kv4(dev(q), dev(pool), dev(pos), layer=1, n_q=n_q, block_table=dev(table), seq=dev(seq), rope_cos=dev(cos), rope_sin=dev(sin), out=out, split_keys=split)
        left = np.setdiff1d(np.arange(len(seq)), refused) if bad else np.arange(len(seq))
        check(host(out)[left], q[left], pool, table, 1, pos[left], seq[left], cos, sin)
        if bad:
            assert (host(out)[refused] == 7.0).all()
        g.check()
        assert kernels.kv4_take_errors() == (2 if bad else 0)


def test_long_rows_that_share_a_sequence(cuda_lib):
    """Drafts of five rows over long contexts: splits joined by clusters and by a second kernel, and keys that only the later rows see."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(77)
    for n_q, n_kv, lens in ((20, 5, [6000, 4096]), (16, 4, [1029, 1024, 900, 1027]), (8, 8, [3000, 2500, 2049])):
        table, pool = setup(rng, lens, n_kv, (max(lens) + 15) // 16)
        seq = np.arange(len(lens), dtype=np.int32).repeat(5)
        pos = np.concatenate([n - 5 + rng.permutation(5) for n in lens]).astype(np.int32)
        q = rng.standard_normal((len(seq), n_q * 128)).astype(np.float32)
        for split in (0, 128, 256):
            out = kernels.attention_kv4(dev(q), dev(pool), dev(pos), layer=0, n_q=n_q, block_table=dev(table), seq=dev(seq), split_keys=split, use_pdl=True)
            check(host(out), q, pool, table, 0, pos, seq)
    assert kernels.kv4_take_errors() == 0


@pytest.mark.parametrize("n_q,n_kv,most,split", [(8, 2, 1000, 0), (20, 5, 9000, 0), (3, 1, 300, 512)])
def test_captured_once_for_growing_sequences(cuda_lib, n_q, n_kv, most, split):
    """A graph captured with one set of lengths and replayed with others, queries and tables changed in place; nothing of an earlier replay stays."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(most)
    columns = (most + 15) // 16
    table, pool = setup(rng, [most, most], n_kv, columns)
    d = dict(q=torch.zeros(2, n_q * 128, device="cuda"), pos=torch.full((2,), most - 1, dtype=torch.int32, device="cuda"), table=dev(table))
    dp = dev(pool)
    call = lambda: kernels.attention_kv4(d["q"], dp, d["pos"], layer=0, n_q=n_q, block_table=d["table"], max_len=most, split_keys=split, use_pdl=True)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for lens in ([1, most], [most // 2, 17], [0, 33], [most, most - 1]):
        q, pos, swapped = rng.standard_normal((2, n_q * 128)).astype(np.float32), np.array(lens, np.int32) - 1, table[::-1].copy()
        for name, x in (("q", q), ("pos", pos), ("table", swapped)):
            d[name].copy_(dev(x))
        graph.replay()
        torch.cuda.synchronize()
        check(host(out), q, pool, swapped, 0, pos, range(2))
    assert kernels.kv4_take_errors() == 0


def test_two_at_once(cuda_lib):
    """Calls on two streams, joined by clusters, by a second kernel, and not at all; each with a workspace of its own."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(31)
    for lens, split in (([900, 1000], 0), ([5000, 4000], 0), ([300, 200], 512)):
        table, pool = setup(rng, lens, 2, (max(lens) + 15) // 16)
        q = [rng.standard_normal((2, 8 * 128)).astype(np.float32) for _ in range(2)]
        pos = np.array(lens, np.int32) - 1
        dq, dp, dpos, dt = [dev(x) for x in q], dev(pool), dev(pos), dev(table)
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        got = [[], []]
        for _ in range(10):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got[i].append(kernels.attention_kv4(dq[i], dp, dpos, layer=0, n_q=8, block_table=dt, split_keys=split, use_pdl=True))
        torch.cuda.synchronize()
        for i in range(2):
            check(host(got[i][0]), q[i], pool, table, 0, pos, range(2))
            assert all(torch.equal(got[i][0], x) for x in got[i])
    assert kernels.kv4_take_errors() == 0


def test_pools_beyond_32_bits(cuda_lib):
    """Blocks whose bytes lie past 2^31 and 2^32 of the pool's start."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(6)
    per_block = 4 * 8 * 2560
    blocks = (2 ** 32 + 2 ** 30) // per_block
    pool = torch.zeros(blocks, 4, 8, 2, 16, 80, dtype=torch.uint8, device="cuda")
    table = np.array([[blocks - 1, 2 ** 31 // per_block + 1, 2 ** 32 // per_block + 1, 0]], np.int32)
    n = 60
    k, v = (rng.standard_normal((n, 8 * 128)).astype(np.float32) for _ in range(2))
    pos = np.arange(n, dtype=np.int32)
    dt, dpos, seq = dev(table), dev(pos), torch.zeros(n, dtype=torch.int32, device="cuda")
    kernels.kv4_append(dev(k), dev(v), pool, dpos, layer=3, block_table=dt, seq=seq)
    rk, rv = kernels.kv4_read(pool, dpos, layer=3, block_table=dt, seq=seq)
    assert np.array_equal(host(rk).reshape(n, 8, 128), ref.values(ref.quantise(k.reshape(n, 8, 128))).astype(np.float32))
    small = host(pool[dt[0].long()])
    q = rng.standard_normal((1, 16 * 128)).astype(np.float32)
    out = kernels.attention_kv4(dev(q), pool, dev(np.array([n - 1], np.int32)), layer=3, n_q=16, block_table=dt)
    check(host(out), q, small, np.arange(4)[None], 3, [n - 1], [0])
    assert kernels.kv4_take_errors() == 0


@pytest.mark.parametrize("splits", [2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("rows,n_q,n_kv", [(2, 4, 1), (3, 3, 1), (1, 5, 5), (2, 20, 5), (2, 7, 1), (40, 8, 1), (45, 7, 1)])
def test_clusters_of_every_size(cuda_lib, rows, n_q, n_kv, splits):
    """Shares of the outputs that no number of warps divides; splits without keys, padding and refused rows beside full ones. (45 rows of 8 splits of seven heads a CTA.)"""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(splits * 100 + n_q)
    most = 128 * splits
    lens = [most] + [int(n) for n in rng.integers(1, most + 1, rows - 1)]
    table, pool = setup(rng, lens, n_kv, most // 16)
    q = rng.standard_normal((rows + 2, n_q * 128)).astype(np.float32)
    seq, pos = np.r_[np.arange(rows), 0, 0].astype(np.int32), np.r_[np.array(lens) - 1, -1, most].astype(np.int32)
    g = Guarded()
    out = g.empty((rows + 2, n_q * 128), torch.float32)
    out.fill_(7.0)
    for pdl in (False, True):
        kernels.attention_kv4(dev(q), dev(pool), dev(pos), layer=0, n_q=n_q, block_table=dev(table), seq=dev(seq), max_len=most, out=out, use_pdl=pdl)
    check(host(out)[:-1], q[:-1], pool, table, 0, pos[:-1], seq[:-1])
    assert (host(out)[-1] == 7.0).all()
    g.check()
    assert kernels.kv4_take_errors() == 2


@pytest.mark.parametrize("n_q,n_kv", [(4, 2), (8, 1)])
def test_values_at_the_ends_of_fp16(cuda_lib, n_q, n_kv):
    """Groups of 65504 alone, of -65504 alone, from one to the other, and clamped ones, as the quantiser leaves them: nothing overflows."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(n_q)
    n, columns = 250, 16
    x = np.clip(rng.standard_normal((columns, 1, n_kv, 2, 16, 128)) * 4e4, -65504, 65504).astype(np.float32)
    x[:, :, :, 0] = rng.standard_normal(x[:, :, :, 0].shape)                # keys of ordinary size
    some = rng.integers(0, 4, (columns, 1, n_kv, 16))
    x[:, :, :, 1][some == 0], x[:, :, :, 1][some == 1] = 65504, -65504
    x[:, :, :, 1, :, 96:] = 65504                                           # a group that no key leaves
    pool, table = ref.quantise(x), rng.permutation(columns).astype(np.int32)[None]
    q, pos = rng.standard_normal((1, n_q * 128)).astype(np.float32), np.array([n - 1], np.int32)
    out = kernels.attention_kv4(dev(q), dev(pool), dev(pos), layer=0, n_q=n_q, block_table=dev(table))
    k, v = ref.cached(pool, 0, table[0], n)
    want, bound = ref.attention(q[0].reshape(n_q, 128), k, v)
    err = abs(host(out)[0].reshape(n_q, 128).astype(np.float64) - want)
    assert (err <= bound).all(), float((err / bound).max())
