"""Rows stored four kv heads a warp, which calls of more than 9472 (row, head) pairs are, bit for bit between guards: heads that no four make up, padding, rows that are refused, rows aligned to
four bytes only, and both sides of the rule."""
import numpy as np
import pytest
import torch
import kv8_reference as ref
from gpu_helpers import dev
from test_gpu_kv8_rows import OnGpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,n_kv,slots,offset", [(2000, 5, 16, 0), (3300, 3, 48, 0), (1300, 8, 16, 0), (1400, 7, 16, 1), (1700, 6, 16, 0), (2500, 4, 2512, 3), (1184, 8, 16, 0), (1185, 8, 16, 0), (1895, 5, 16, 2)])
def test_many_rows(cuda_lib, rows, n_kv, slots, offset):
    from tenzo_b200 import kernels
    rng = np.random.default_rng(rows + n_kv)
    n_seq, layers, layer, start = 3, 2, 1, 5
    tokens = (rows + n_seq - 1) // n_seq
    c = ref.Caches(rng, n_seq, (start + tokens + slots - 1) // slots, layers, n_kv, slots)
    seq, place = (np.arange(rows) % n_seq).astype(np.int32), (start + np.arange(rows) // n_seq).astype(np.int32)
    order = rng.permutation(rows)
    seq, place = seq[order], place[order]
    pos = (place + rng.integers(0, 50, rows)).astype(np.int32)
    length = int(pos.max()) + 1
    cos, sin = ref.rope(length)
    place[rng.random(rows) < 0.1] = -1
    bad = rng.choice(np.flatnonzero(place >= 0), 5, replace=False)             # beyond the table, no such table rows, no such positions
    place[bad[0]], seq[bad[1]], seq[bad[2]], pos[bad[3]], pos[bad[4]] = c.table.shape[1] * slots, n_seq, -1, length, -1
    gone = (1, (start + tokens // 2) // slots)                                  # and an entry of the table that is none
    kept = c.table.copy()
    if slots < 100:
        c.table[gone] = c.n_blocks
    wide = [(rng.standard_normal((rows, offset + n_kv * 128 + 4 - offset)) * 3).astype(np.float32) for _ in range(2)]
    k, v = (x[:, offset: offset + n_kv * 128] for x in wide)
    g = OnGpu(c)
    kernels.kv8_append(*(dev(x)[:, offset: offset + n_kv * 128] for x in wide), g.cache, dev(place), layer=layer, seq=dev(seq), rope_pos=dev(pos), rope_cos=dev(cos), rope_sin=dev(sin),
                       weight=g.weight, position=g.position)
    there = place >= 0
    there[bad] = False
    if slots < 100:
        there &= ~((seq == gone[0]) & (np.maximum(place, 0) // slots == gone[1]))
        assert not there.all() and kept[gone] != c.table[gone]
    i = np.flatnonzero(there)
    b, o = c.at(seq[i], place[i])
    turn = [x[pos[i]][:, None] for x in (cos, sin)]
    for x, codes, scales, turned in ((k, c.k, c.sk, True), (v, c.v, c.sv, False)):
        x = x[i].reshape(len(i), n_kv, 128)
        codes[b, layer, :, o], scales[b, layer, :, o] = ref.quantise(ref.rotate32(x, *turn) if turned else x)
    c.weight[b, layer, :, o], c.position[b, layer, :, o] = 0, pos[i][:, None]
    g.check(c)
    assert kernels.kv8_take_errors() == 2
