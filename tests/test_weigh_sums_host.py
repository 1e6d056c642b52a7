"""The sums that kv8_weigh adds to the weights at the end of a block of tiles, run on the host: they come to the rows that are remembered, and after a wait that
was given up, when neither rows nor sums need have been written, no weight is touched."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    from tenzo_b200.build import nvcc_path
    out = tmp_path_factory.mktemp("weigh") / "libweigh_host.so"
    r = subprocess.run([nvcc_path(), "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-Xcompiler", "-fPIC", "-shared", str(ROOT / "tests" / "host" / "weigh_sums_host.cu"), "-o", str(out)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    return C.CDLL(str(out))


SHAPES = {3: (42, 50), 4: (32, 40)}               # queries by sixteen: tiles of a block, and tiles whose rows are remembered


def call(lib, groups, given_up, n, t0, t1, total, rows, sums, weight):
    lib.weigh_add_host(groups, int(given_up), n, t0, t1, total, rows.ctypes.data_as(C.c_void_p), sums.ctypes.data_as(C.c_void_p), weight.ctypes.data_as(C.c_void_p))


@pytest.mark.parametrize("groups", [3, 4])
@pytest.mark.parametrize("t0,tiles,n,total", [(0, 1, 1, 1), (0, 3, 3, 300), (7, 5, 61, 12 * 128 - 100), (2, 32, 133, 34 * 128)])
def test_sums_come_to_their_rows(lib, groups, t0, tiles, n, total):
    most, remembered = SHAPES[groups]
    rng = np.random.default_rng(n)
    rows = np.full((remembered, 8), 1 << 30, np.int32)                         # of tiles that are not this block's: not to be looked at
    chunks = rng.permutation(tiles * 8 + 5)[: tiles * 8].reshape(tiles, 8) * 16
    chunks[0, 1:][rng.random(7) < 0.3] = -1
    for i in range(tiles):
        rows[(n - tiles + i) % remembered] = chunks[i]
    sums = rng.integers(0, 9, (groups, most, 128)).astype(np.float32)
    weight = rng.integers(0, 9, (tiles * 8 + 5) * 16).astype(np.float32)
    want = weight.copy()
    for k in range(tiles * 128):
        row = chunks[k // 128, k % 128 // 16]
        if row >= 0 and t0 * 128 + k < total:
            want[row + k % 16] += sums[:, k // 128, k % 128].sum()
    call(lib, groups, False, n, t0, t0 + tiles, total, rows, sums, weight)
    assert np.array_equal(weight, want)


@pytest.mark.parametrize("groups", [3, 4])
def test_nothing_is_touched_after_a_wait_was_given_up(lib, groups):
    most, remembered = SHAPES[groups]
    weight = np.arange(4096, dtype=np.float32)
    call(lib, groups, True, 9, 0, 9, 9 * 128, np.full((remembered, 8), 64, np.int32), np.full((groups, most, 128), np.nan, np.float32), weight)
    assert np.array_equal(weight, np.arange(4096))
