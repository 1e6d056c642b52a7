"""Rows of the 4-bit paged cache on the GPU: appended bytes and read-back values are the definition's, bit for bit, and no other byte changes."""
import numpy as np
import pytest
import torch
import kv4_reference as ref
from gpu_helpers import Guarded, dev, host

pytestmark = pytest.mark.gpu


def setup(rng, n_seq, columns, layers, n_kv):
    blocks = n_seq * columns + 3
    table = rng.permutation(blocks)[: n_seq * columns].astype(np.int32).reshape(n_seq, columns)
    pool = rng.integers(0, 256, (blocks, layers, n_kv, 2, 16, 80), dtype=np.uint8)       # what lies there is anything, NaN among it
    return table, pool


def expect(pool, table, layer, k, v, pos, seq, cos, sin):
    pool, n_kv = pool.copy(), pool.shape[2]
    for i, (p, s) in enumerate(zip(pos, seq)):
        if p < 0:
            continue
        key = k[i].reshape(n_kv, 128)
        if cos is not None:
            key = ref.rotate(key, cos[p], sin[p])
        block = table[s, p // 16]
        pool[block, layer, :, 0, p % 16] = ref.quantise(key)
        pool[block, layer, :, 1, p % 16] = ref.quantise(v[i].reshape(n_kv, 128))
    return pool


@pytest.mark.parametrize("n_seq,tokens,start,n_kv,layers,layer,rotated,padded", [
    (1, 1, 0, 5, 1, 0, True, False),
    (3, 1, 15, 1, 2, 1, True, False),
    (2, 37, 11, 5, 3, 1, True, True),
    (5, 16, 16, 8, 1, 0, False, False),
    (1, 133, 0, 2, 1, 0, True, False),
    (64, 1, 200, 5, 2, 0, True, True),
])
def test_append_and_read(cuda_lib, n_seq, tokens, start, n_kv, layers, layer, rotated, padded):
    from tenzo_b200 import kernels
    rng = np.random.default_rng(n_seq * 1000 + tokens)
    columns = (start + tokens + 15) // 16
    table, pool = setup(rng, n_seq, columns, layers, n_kv)
    seq = np.repeat(np.arange(n_seq), tokens).astype(np.int32)
    pos = np.tile(start + np.arange(tokens), n_seq).astype(np.int32)
    order = rng.permutation(len(pos))                                       # rows come in any order
    seq, pos = seq[order], pos[order]
    if padded:
        pos[rng.random(len(pos)) < 0.3] = -1
    k, v = (rng.standard_normal((len(pos), n_kv * 128)).astype(np.float32) * 3 for _ in range(2))
    cos, sin = ref.rope(start + tokens) if rotated else (None, None)
    g = Guarded()
    d_pool = g.empty(pool.shape, torch.uint8, dev(pool))
    tables = dict(rope_cos=dev(cos), rope_sin=dev(sin)) if rotated else {}
    kernels.kv4_append(dev(k), dev(v), d_pool, dev(pos), layer=layer, block_table=dev(table), seq=dev(seq), **tables)
    want = expect(pool, table, layer, k, v, pos, seq, cos, sin)
    got = host(d_pool)
    assert np.array_equal(got, want)
    rk, rv = kernels.kv4_read(d_pool, dev(pos), layer=layer, block_table=dev(table), seq=dev(seq))
    stored = ref.values(want[table[seq, np.maximum(pos, 0) // 16], layer, :, :, np.maximum(pos, 0) % 16])     # [rows, heads, 2, 128]
    stored[pos < 0] = 0
    assert np.array_equal(host(rk), stored[:, :, 0].reshape(len(pos), -1).astype(np.float32))       # one rounding, of the sum
    assert np.array_equal(host(rv), stored[:, :, 1].reshape(len(pos), -1).astype(np.float32))
    g.check()
    assert kernels.kv4_take_errors() == 0


@pytest.mark.parametrize("offset", [0, 1, 4])
def test_rows_of_a_wider_buffer(cuda_lib, offset):
    """k and v as column slices of a q|k|v buffer, also where their rows do not start at 16 bytes; read into such a buffer."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(offset)
    n, n_kv = 21, 3
    table, pool = setup(rng, n, 2, 1, n_kv)
    wide = rng.standard_normal((n, 1000 + offset)).astype(np.float32)
    d = dev(wide)
    pos = rng.integers(0, 32, n).astype(np.int32)
    d_pool, d_table = dev(pool), dev(table)
    kernels.kv4_append(d[:, offset: offset + 384], d[:, 500 + offset: 884 + offset], d_pool, dev(pos), layer=0, block_table=d_table)
    want = expect(pool, table, 0, wide[:, offset: offset + 384], wide[:, 500 + offset: 884 + offset], pos, range(n), None, None)
    assert np.array_equal(host(d_pool), want)
    back = torch.full((n, 1000 + offset), 7.0, device="cuda")
    kernels.kv4_read(d_pool, dev(pos), layer=0, block_table=d_table, k=back[:, offset: offset + 384], v=back[:, 500 + offset: 884 + offset])
    k, v = kernels.kv4_read(d_pool, dev(pos), layer=0, block_table=d_table)
    assert torch.equal(back[:, offset: offset + 384], k) and torch.equal(back[:, 500 + offset: 884 + offset], v)
    assert bool((back[:, :offset] == 7).all()) and bool((back[:, 384 + offset: 500 + offset] == 7).all()) and bool((back[:, 884 + offset:] == 7).all())


def test_values_at_the_quantisers_edges(cuda_lib):
    """Constant groups, zeros of both signs, one outlier, ranges below fp16's smallest step, numbers fp16 cannot hold, codes half way between two."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(5)
    groups = [np.full(32, 2.5), np.zeros(32), np.where(np.arange(32) % 2, -0.0, 0.0), np.r_[1000.0, rng.standard_normal(31) * 1e-3],
              1.0 + rng.standard_normal(32) * 1e-8, rng.standard_normal(32) * 1e-7, rng.standard_normal(32) * 1e-30, rng.standard_normal(32) * 1e6,
              np.r_[-3e38, 3e38, np.zeros(30)], np.arange(32) / 2.0 % 15.0, np.r_[0.0, 15.0, np.arange(30) / 2.0], -np.arange(32) * 65504 / 31,
              rng.standard_normal(32) * 2000, np.r_[0.0, 2.0 ** -24 * 15, np.zeros(30)], np.full(32, 65519.9), np.full(32, 1e-8)]
    x = np.stack(groups).astype(np.float32).reshape(-1, 128)
    n = len(x)
    pool = np.zeros((n, 1, 1, 2, 16, 80), np.uint8)
    table = np.arange(n, dtype=np.int32)[:, None]
    d = dev(pool)
    kernels.kv4_append(dev(x), dev(-x), d, dev(np.full(n, 3, np.int32)), layer=0, block_table=dev(table))
    got = host(d)
    # a zero minimum may carry either sign
    canon = lambda rows: np.where(rows.view(np.uint16) == 0x8000, 0, rows.view(np.uint16)) if rows.shape[-1] == 16 else rows    # noqa: E731
    for i, want in ((0, ref.quantise(x)), (1, ref.quantise(-x))):
        assert np.array_equal(got[:, 0, 0, i, 3, :64], want[:, :64])
        assert np.array_equal(canon(np.ascontiguousarray(got[:, 0, 0, i, 3, 64:])), canon(np.ascontiguousarray(want[:, 64:])))
    k, v = kernels.kv4_read(d, dev(np.full(n, 3, np.int32)), layer=0, block_table=dev(table))
    assert bool(torch.isfinite(k).all()) and bool(torch.isfinite(v).all())
    # off by half a step and the parameters' own rounding at most: the minimum's half step (2^-11 of it) and 15 times the scale's
    lo, hi = np.clip(x, -65504, 65504).reshape(-1, 32).min(1), np.clip(x, -65504, 65504).reshape(-1, 32).max(1)
    err = abs(host(k).reshape(-1, 32).astype(np.float64) - np.clip(x, -65504, 65504).reshape(-1, 32)).max(1)
    room = (hi.astype(np.float64) - lo + abs(lo) * 2.0 ** -11) / 30 * (1 + 2.0 ** -9) + abs(lo) * 2.0 ** -11 + (hi.astype(np.float64) - lo) * 2.0 ** -10 + 16 * 2.0 ** -25
    assert (err <= room).all(), (err, room)


def test_non_finite_values_stay_in_their_group(cuda_lib):
    from tenzo_b200 import kernels
    x = np.random.default_rng(1).standard_normal((2, 128)).astype(np.float32)
    bad = x.copy()
    bad[0, 40], bad[0, 70], bad[1, 3] = np.nan, np.inf, -np.inf
    out = []
    for rows in (x, bad):
        d = torch.zeros(2, 1, 1, 2, 16, 80, dtype=torch.uint8, device="cuda")
        table = torch.arange(2, dtype=torch.int32, device="cuda")[:, None].contiguous()
        pos = torch.zeros(2, dtype=torch.int32, device="cuda")
        kernels.kv4_append(dev(rows), dev(rows), d, pos, layer=0, block_table=table)
        out.append(host(kernels.kv4_read(d, pos, layer=0, block_table=table)[0]).reshape(2, 4, 32))
    clean = np.ones((2, 4), bool)
    clean[0, 1] = clean[0, 2] = clean[1, 0] = False
    assert np.array_equal(out[0][clean], out[1][clean]) and np.isfinite(out[1]).all()


def test_indices_out_of_range_touch_nothing(cuda_lib):
    from tenzo_b200 import kernels
    rng = np.random.default_rng(9)
    table, pool = setup(rng, 4, 2, 1, 2)
    table[2, 1], table[3, 0] = len(pool), -1
    k, v = (rng.standard_normal((8, 256)).astype(np.float32) for _ in range(2))
    #           fine     past the table   no such sequence   block too large, negative   past the rotation's tables, padding
    seq = np.array([0, 1, 1, 4, -1, 2, 3, 0], np.int32)
    pos = np.array([3, 31, 32, 0, 0, 17, 5, -7], np.int32)
    cos, sin = ref.rope(32)
    assert kernels.kv4_take_errors() == 0
    g = Guarded()
    d_pool = g.empty(pool.shape, torch.uint8, dev(pool))
    kernels.kv4_append(dev(k), dev(v), d_pool, dev(pos), layer=0, block_table=dev(table), seq=dev(seq), rope_cos=dev(cos), rope_sin=dev(sin))
    assert kernels.kv4_take_errors() == 2 and kernels.kv4_take_errors() == 0
    good = np.where(np.arange(8) < 2, pos, -1)
    assert np.array_equal(host(d_pool), expect(pool, table, 0, k, v, good, np.clip(seq, 0, 3), cos, sin))
    rk, _ = kernels.kv4_read(d_pool, dev(pos), layer=0, block_table=dev(table), seq=dev(seq))
    assert kernels.kv4_take_errors() == 2
    assert bool((rk[2:] == 0).all()) and bool((rk[:2] != 0).any())
    kernels.kv4_append(dev(k), dev(v), d_pool, dev(np.array([-1, 20, -1, -1, -1, -1, -1, -1], np.int32)), layer=0, block_table=dev(table), seq=dev(seq), rope_cos=dev(cos[:20]),
                       rope_sin=dev(sin[:20]))
    assert kernels.kv4_take_errors() == 2
    assert np.array_equal(host(d_pool), expect(pool, table, 0, k, v, good, np.clip(seq, 0, 3), cos, sin))
    g.check()


def test_no_rows(cuda_lib):
    from tenzo_b200 import kernels
    pool = torch.zeros(2, 1, 1, 2, 16, 80, dtype=torch.uint8, device="cuda")
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    none, pos = torch.empty(0, 128, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda")
    kernels.kv4_append(none, none, pool, pos, layer=0, block_table=table)
    k, v = kernels.kv4_read(pool, pos, layer=0, block_table=table)
    assert k.shape == v.shape == (0, 128)
    assert kernels.attention_kv4(none, pool, pos, layer=0, n_q=1, block_table=table).shape == (0, 128)


def test_on_a_side_stream_and_in_a_graph(cuda_lib):
    from tenzo_b200 import kernels
    rng = np.random.default_rng(3)
    table, pool = setup(rng, 6, 3, 1, 2)
    k, v, pos = rng.standard_normal((6, 256)).astype(np.float32), rng.standard_normal((6, 256)).astype(np.float32), rng.integers(0, 48, 6).astype(np.int32)
    want = expect(pool, table, 0, k, v, pos, range(6), None, None)
    dk, dv, dp, dt, d = dev(k), dev(v), dev(pos), dev(table), dev(pool)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kernels.kv4_append(dk, dv, d, dp, layer=0, block_table=dt)
        first = kernels.kv4_read(d, dp, layer=0, block_table=dt)
    side.synchronize()
    assert np.array_equal(host(d), want)
    d.copy_(dev(pool))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kernels.kv4_append(dk, dv, d, dp, layer=0, block_table=dt, use_pdl=True)
        second = kernels.kv4_read(d, dp, layer=0, block_table=dt, use_pdl=True)
    d.copy_(dev(pool))
    graph.replay()
    assert np.array_equal(host(d), want) and all(torch.equal(a, b) for a, b in zip(first, second))
    dk.add_(1.0)                                                            # a replay works on what the tensors hold then
    d.copy_(dev(pool))
    graph.replay()
    assert np.array_equal(host(d), expect(pool, table, 0, k + np.float32(1), v, pos, range(6), None, None))


def test_errors_of_a_stream_that_is_still_running(cuda_lib):
    """The query waits for streams that do not wait for the default stream, and reports what was raised there; each flag once."""
    from tenzo_b200 import kernels
    pool, table = torch.zeros(2, 1, 1, 2, 16, 80, dtype=torch.uint8, device="cuda"), torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    rows, beyond = torch.ones(1, 128, device="cuda"), torch.full((1,), 16, dtype=torch.int32, device="cuda")
    calls = [lambda: kernels.kv4_append(rows, rows, pool, beyond, layer=0, block_table=table),
             lambda: kernels.attention_kv4(rows, pool, beyond, layer=0, n_q=1, block_table=table, out=torch.empty_like(rows))]
    for call in calls:                                                      # (both modules loaded before the query is to be quicker than the stream)
        call()
    torch.cuda.synchronize()
    assert kernels.kv4_take_errors() == 2
    for call in calls:
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            torch.cuda._sleep(200_000_000)                                  # about 0.1 s
            call()
        assert kernels.kv4_take_errors() == 2
        assert kernels.kv4_take_errors() == 0


@pytest.mark.parametrize("n,n_kv,rotated,offset,broken", [
    (1185, 8, True, 0, False), (1185, 8, True, 1, True), (9473, 1, True, 0, True), (9473, 1, False, 2, False), (2049, 5, False, 0, True), (9472, 1, True, 4, False), (4001, 3, True, 3, True),
])
def test_many_rows(cuda_lib, n, n_kv, rotated, offset, broken):
    """As many rows and heads as two rows a warp are taken for: odd numbers of them; padding, and indices out of range, in either half of a pair and in the last row; rows of wider buffers, whether they
    start at 16 bytes or not."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(n + offset)
    assert n * n_kv >= 9472
    n_seq, columns = 37, n // 37 // 16 + 2
    table, pool = setup(rng, n_seq, columns, 2, n_kv)
    place = rng.permutation(n_seq * columns * 16)[:n]    # no token twice
    seq, pos = (place // (columns * 16)).astype(np.int32), (place % (columns * 16)).astype(np.int32)
    pos[rng.random(n) < 0.2] = -1
    want_pos, cos, sin = pos.copy(), *ref.rope(columns * 16)
    if broken:
        bad = rng.choice(n, n // 10, replace=False)
        bad[0] = n - 1
        for i, r in enumerate(bad):                      # past the table, no such sequence
            seq[r], pos[r] = [(0, columns * 16), (n_seq, 3), (-1, 0), (1 << 30, 1 << 30)][i % 4]
        want_pos[bad] = -1
        table[5, :] = [-1 if c % 2 else len(pool) for c in range(columns)]
        want_pos[seq == 5] = -1
    width = n_kv * 128
    wide = rng.standard_normal((n, 2 * width + 8 + offset)).astype(np.float32) * 3
    k, v = wide[:, offset: offset + width], wide[:, offset + width + 4: offset + 4 + 2 * width]
    d = dev(wide)
    g = Guarded()
    d_pool = g.empty(pool.shape, torch.uint8, dev(pool))
    rope = dict(rope_cos=dev(cos), rope_sin=dev(sin)) if rotated else {}
    kernels.kv4_append(d[:, offset: offset + width], d[:, offset + width + 4: offset + 4 + 2 * width], d_pool, dev(pos), layer=1, block_table=dev(table), seq=dev(seq), **rope)
    rows = np.flatnonzero(want_pos >= 0)
    keys = k.reshape(n, n_kv, 128)[rows]
    if rotated:
        keys = ref.rotate(keys, cos[want_pos[rows]][:, None], sin[want_pos[rows]][:, None])
    want = pool.copy()
    block, slot = table[seq[rows], want_pos[rows] // 16], want_pos[rows] % 16
    want[block, 1, :, 0, slot], want[block, 1, :, 1, slot] = ref.quantise(keys), ref.quantise(v.reshape(n, n_kv, 128)[rows])
    assert np.array_equal(host(d_pool), want)
    assert kernels.kv4_take_errors() == (2 if broken else 0)
    back = [g.empty((n, width), torch.float32) for _ in range(2)]
    for to in back:
        to.fill_(7.0)
    apart = torch.full((n, 2 * width + 8 + offset), 7.0, device="cuda")
    kernels.kv4_read(d_pool, dev(pos), layer=1, block_table=dev(table), seq=dev(seq), k=back[0], v=back[1])
    kernels.kv4_read(d_pool, dev(pos), layer=1, block_table=dev(table), seq=dev(seq), k=apart[:, offset: offset + width], v=apart[:, offset + width + 4: offset + 4 + 2 * width], use_pdl=True)
    stored = np.zeros((n, n_kv, 2, 128))
    stored[rows] = ref.values(want[block, 1, :, :, slot])
    for i, at in enumerate((offset, offset + width + 4)):
        assert np.array_equal(host(back[i]), stored[:, :, i].reshape(n, -1).astype(np.float32))
        assert torch.equal(apart[:, at: at + width], back[i])
        apart[:, at: at + width] = 7.0
    assert bool((apart == 7.0).all())
    assert kernels.kv4_take_errors() == (2 if broken else 0)
    g.check()
