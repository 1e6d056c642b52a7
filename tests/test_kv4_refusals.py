"""What the 4-bit cache's and the beam selection's entry points refuse, without a device: refusals come before any launch. And the packed
arguments of the Python calls are the C structs."""
import ctypes as C

import pytest
import torch
from tenzo_b200 import abi, kernels, load_library

P = 0x10000                                       # a 16-byte aligned address that nothing looks at


@pytest.fixture(scope="module")
def lib():
    return load_library()


def cache(**over):
    c = abi.Kv4Cache(pool=P, n_blocks=10, n_layers=2, n_kv=3, block_table=P, table_rows=4, table_stride=5)
    for k, v in over.items():
        setattr(c, k, v)
    return c


BAD_CACHES = [dict(pool=None), dict(pool=P + 8), dict(block_table=None), dict(n_blocks=0), dict(n_layers=0), dict(n_kv=0), dict(table_rows=0), dict(table_stride=0)]


@pytest.mark.parametrize("over", BAD_CACHES, ids=str)
def test_caches(lib, over):
    c = cache(**over)
    assert lib.tenzo_cuda_kv4_append(C.byref(c), 0, P, P, 384, P, P, 4, None, None, 0, 0, None) == abi.ERR_INVALID
    assert lib.tenzo_cuda_kv4_read(C.byref(c), 0, P, P, 384, P, P, 4, 0, None) == abi.ERR_INVALID
    assert lib.tenzo_cuda_kv4_reorder(C.byref(c), P + 64, P, P, 2, 2, 0, None) == abi.ERR_INVALID
    assert lib.tenzo_cuda_attention_kv4(C.byref(attention(cache=c)), None) == abi.ERR_INVALID


@pytest.mark.parametrize("change", [dict(layer=-1), dict(layer=2), dict(k=None), dict(v=None), dict(stride=383), dict(pos=None), dict(rows=-1), dict(seq=None, rows=5),
                                    dict(cos=P), dict(sin=P), dict(cos=P, sin=P, length=0)], ids=str)
def test_append(lib, change):
    a = dict(layer=0, k=P, v=P, stride=384, pos=P, seq=P, rows=4, cos=None, sin=None, length=0) | change
    assert lib.tenzo_cuda_kv4_append(C.byref(cache()), a["layer"], a["k"], a["v"], a["stride"], a["pos"], a["seq"], a["rows"], a["cos"], a["sin"], a["length"], 0,
                                     None) == abi.ERR_INVALID


@pytest.mark.parametrize("change", [dict(layer=-1), dict(layer=2), dict(k=None, v=None), dict(stride=383), dict(pos=None), dict(rows=-1), dict(seq=None, rows=5)], ids=str)
def test_read(lib, change):
    a = dict(layer=0, k=P, v=P, stride=384, pos=P, seq=P, rows=4) | change
    assert lib.tenzo_cuda_kv4_read(C.byref(cache()), a["layer"], a["k"], a["v"], a["stride"], a["pos"], a["seq"], a["rows"], 0, None) == abi.ERR_INVALID


def attention(**over):
    a = abi.AttentionKv4Args(q=P, out=P, cache=cache(), pos=P, seq=P, layer=0, n_q=6, rows=4, max_len=80)
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over", [dict(q=None), dict(out=None), dict(pos=None), dict(layer=2), dict(layer=-1), dict(n_q=0), dict(n_q=7), dict(rows=-1), dict(max_len=0),
                                  dict(max_len=81), dict(max_len=(1 << 30) + 1), dict(seq=None, rows=5), dict(rope_cos=P), dict(rope_sin=P), dict(rope_cos=P, rope_sin=P, rope_len=79),
                                  dict(q_stride=767), dict(split_keys=-1), dict(out=P + 4), dict(split_keys=16), dict(split_keys=16, workspace=P + 8, workspace_bytes=1 << 30),
                                  dict(split_keys=16, max_len=80, workspace=P, workspace_bytes=10)], ids=str)
def test_attention(lib, over):
    if over.get("max_len") == (1 << 30) + 1:
        over = dict(over, cache=cache(table_stride=1 << 27))
    if "split_keys" in over and over["split_keys"] == 16:
        over = dict(over, cache=cache(table_stride=100), max_len=1000)       # eight splits, and no room for them
    assert lib.tenzo_cuda_attention_kv4(C.byref(attention(**over)), None) == abi.ERR_INVALID


def test_attention_null_and_sizes(lib):
    assert lib.tenzo_cuda_attention_kv4(None, None) == abi.ERR_INVALID
    need = lib.tenzo_cuda_attention_kv4_workspace_bytes
    assert need(0, 4, 2, 10) == need(1, 0, 2, 10) == need(1, 4, 0, 10) == need(1, 5, 2, 10) == need(1, 4, 2, 0) == 0
    assert need(64, 20, 5, 8192) < need(128, 20, 5, 8192) and need(1, 4, 2, 1) > 0


def test_attention_room_for_the_chosen_splits(lib):
    splits = lib.tenzo_cuda_attention_kv4_splits
    assert splits(0, 4, 2, 10) == splits(1, 0, 2, 10) == splits(1, 4, 0, 10) == splits(1, 5, 2, 10) == splits(1, 4, 2, 0) == splits(1, 4, 2, (1 << 30) + 1) == 0
    assert splits(1, 20, 5, 100) == splits(1, 20, 5, 1000) == 1 and splits(1, 20, 5, 16384) > 8             # no room for one split, nor for a cluster's
    for rows, n_q, n_kv, n in ((1, 40, 5, 16384), (64, 20, 5, 8192), (256, 20, 5, 131072), (3, 7, 1, 1 << 30), (100000, 32, 32, 4096)):
        most = splits(rows, n_q, n_kv, n)
        assert 1 <= most <= 64 and most * rows * n_q * 520 <= max(lib.tenzo_cuda_attention_kv4_workspace_bytes(rows, n_q, n_kv, n), rows * n_q * 520)
        assert kernels._attention_kv4_room(rows, n_q, n_kv, n, 0) == (most * rows * n_q * 520 if most > 1 else 0)
    assert kernels._attention_kv4_room(2, 4, 2, 1000, 128) == 8 * 2 * 4 * 520 and kernels._attention_kv4_room(2, 4, 2, 1000, 900) == 0       # 900: rounded up to 1024


@pytest.mark.parametrize("change,code", [(dict(out=None), -1), (dict(out=P), -1), (dict(parent=None), -1), (dict(length=None), -1), (dict(groups=0), -1), (dict(groups=-2), -1),
                                         (dict(groups=3), -1), (dict(beams=0), -5), (dict(beams=33), -5), (dict(layers=10000), -5)], ids=str)
def test_reorder(lib, change, code):
    a = dict(out=P + 4096, parent=P, length=P, groups=2, beams=2, layers=2) | change
    assert lib.tenzo_cuda_kv4_reorder(C.byref(cache(n_layers=a["layers"])), a["out"], a["parent"], a["length"], a["groups"], a["beams"], 0, None) == code
    assert lib.tenzo_cuda_kv4_reorder(None, P, P, P, 2, 2, 0, None) == -1


@pytest.mark.parametrize("over,code", [(dict(logits=None), -1), (dict(scores=None), -1), (dict(parent_out=None), -1), (dict(token_out=None), -1), (dict(score_out=None), -1),
                                       (dict(workspace=None), -1), (dict(workspace=P + 4), -1), (dict(workspace_bytes=8), -1), (dict(groups=-1), -1), (dict(beams=0), -1), (dict(beams=33), -5),
                                       (dict(vocab=0), -1), (dict(k=0), -1), (dict(k=65), -5), (dict(vocab=3, k=7), -1), (dict(row_stride=99), -1), (dict(finished=P, eos=100), -1),
                                       (dict(finished=P, eos=-1), -1)], ids=str)
def test_select(lib, over, code):
    a = abi.BeamSelectArgs(logits=P, scores=P, groups=3, beams=2, vocab=100, k=4, parent_out=P, token_out=P, score_out=P, workspace=P, workspace_bytes=1 << 20)
    for k, v in over.items():
        setattr(a, k, v)
    assert lib.tenzo_cuda_beam_select(C.byref(a), None) == code
    assert lib.tenzo_cuda_beam_select(None, None) == -1


def test_nothing_to_do_is_no_error(lib):
    assert lib.tenzo_cuda_kv4_append(C.byref(cache()), 0, None, None, 384, None, None, 0, None, None, 0, 0, None) == 0
    assert lib.tenzo_cuda_kv4_read(C.byref(cache()), 0, None, None, 384, None, None, 0, 0, None) == 0
    assert lib.tenzo_cuda_attention_kv4(C.byref(attention(rows=0, q=None)), None) == 0
    assert lib.tenzo_cuda_beam_select(C.byref(abi.BeamSelectArgs(groups=0)), None) == 0


def _leaves(cls):
    return [x for _, t in cls._fields_ for x in (_leaves(t) if issubclass(t, C.Structure) else [t])]


def _flat(o):
    return [x for n, t in o._fields_ for x in (_flat(getattr(o, n)) if issubclass(t, C.Structure) else [getattr(o, n)])]


@pytest.mark.parametrize("packed,cls", [(kernels._KV4_CACHE, abi.Kv4Cache), (kernels._KV4_ATTENTION, abi.AttentionKv4Args), (kernels._BEAM_SELECT, abi.BeamSelectArgs)])
def test_packed_arguments_are_the_structs(packed, cls):
    numbers = list(range(1, len(_leaves(cls)) + 1))
    assert _flat(cls.from_buffer_copy(packed.pack(*numbers))) == numbers


def test_c_header_layout(tmp_path):
    import subprocess
    from pathlib import Path
    names = [("tenzo_kv4_cache", abi.Kv4Cache, "table_stride"), ("tenzo_attention_kv4_args", abi.AttentionKv4Args, "workspace_bytes"),
             ("tenzo_beam_select_args", abi.BeamSelectArgs, "workspace_bytes")]
    src = tmp_path / "probe.c"
    src.write_text('#include <stdio.h>\n#include "tenzo_kernels.h"\nint main(){' + "".join(
        f'printf("%zu %zu ", sizeof({n}), offsetof({n}, {last}));' for n, _, last in names) + "return 0;}")
    subprocess.run(["gcc", "-I", str(Path(__file__).resolve().parents[1] / "include"), str(src), "-o", str(tmp_path / "probe")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "probe")], capture_output=True, text=True).stdout.split()]
    assert got == [x for _, cls, last in names for x in (C.sizeof(cls), getattr(cls, last).offset)]


def test_python_calls_refuse_tensors_of_the_host():
    """Every tensor has to lie on the current device, in the type and layout that the kernels read."""
    pool, table, pos = torch.zeros(4, 1, 1, 2, 16, 80, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    rows = torch.zeros(2, 128)
    for call in (lambda: kernels.kv4_append(rows, rows, pool, pos, layer=0, block_table=table), lambda: kernels.kv4_read(pool, pos, layer=0, block_table=table),
                 lambda: kernels.attention_kv4(rows, pool, pos, layer=0, n_q=1, block_table=table), lambda: kernels.beam_select(rows, torch.zeros(2), beams=2, k=2),
                 lambda: kernels.kv4_reorder(pool, table, torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))):
        with pytest.raises(Exception) as e:
            call()
        assert isinstance(e.value, (ValueError, RuntimeError))


def test_python_calls_refuse_what_does_not_fit(monkeypatch):
    monkeypatch.setattr(kernels, "_current_device", lambda: -1)              # where the host's tensors lie; nothing gets as far as a launch
    pool, table, pos = torch.zeros(4, 1, 1, 2, 16, 80, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    rows, scores = torch.zeros(2, 128), torch.zeros(2)
    for call in (lambda: kernels.kv4_read(pool, pos, layer=0, block_table=table, k=rows), lambda: kernels.kv4_read(pool, pos, layer=0, block_table=table, v=rows),
                 lambda: kernels.kv4_read(pool, pos, layer=0, block_table=table, k=rows[:1], v=rows[:1]), lambda: kernels.kv4_append(rows, rows[:1], pool, pos, layer=0, block_table=table),
                 lambda: kernels.kv4_append(rows, rows, pool, pos[:1], layer=0, block_table=table), lambda: kernels.kv4_append(rows.double(), rows, pool, pos, layer=0, block_table=table),
                 lambda: kernels.kv4_append(rows, rows, pool.view(4, 1, 1, 2, 80, 16), pos, layer=0, block_table=table),
                 lambda: kernels.attention_kv4(rows, pool, pos, layer=0, n_q=2, block_table=table), lambda: kernels.attention_kv4(rows, pool, pos.long(), layer=0, n_q=1, block_table=table),
                 lambda: kernels.attention_kv4(rows, pool, pos, layer=0, n_q=1, block_table=table, rope_cos=torch.zeros(32, 64)),
                 lambda: kernels.beam_select(rows, scores, beams=0, k=2), lambda: kernels.beam_select(rows, scores, beams=-1, k=2), lambda: kernels.beam_select(rows, scores, beams=2, k=0),
                 lambda: kernels.attention_kv4(rows[:1].expand(2, 128), pool, pos, layer=0, n_q=1, block_table=table), lambda: kernels.beam_select(rows[:1].expand(2, 128), scores, beams=2, k=2),
                 lambda: kernels.kv4_append(rows, rows[:1].expand(2, 128), pool, pos, layer=0, block_table=table), lambda: kernels.attention_kv4(rows[0], pool, pos, layer=0, n_q=1, block_table=table),
                 lambda: kernels.beam_select(rows.flatten().unfold(0, 128, 64), torch.zeros(3), beams=3, k=2), lambda: kernels.beam_select(rows[0], scores, beams=1, k=2),
                 lambda: kernels.beam_select(rows[:1], scores[:1], beams=2, k=2), lambda: kernels.beam_select(rows.half(), scores, beams=2, k=2),
                 lambda: kernels.beam_select(rows, scores, beams=2, k=2, finished=pos[:1]), lambda: kernels.beam_select(rows.t(), scores, beams=2, k=2),
                 lambda: kernels.kv4_reorder(pool, table, torch.zeros(1, 3, dtype=torch.int32), pos[:1]), lambda: kernels.kv4_reorder(pool, table, torch.zeros(1, 2, dtype=torch.int32), pos)):
        with pytest.raises(ValueError):
            call()


def test_numbers_beyond_a_c_int(monkeypatch):
    """A layer or a distance of rows of 2^32 and something is refused, not taken modulo 2^32; how far from the next the only row would lie does not matter."""
    monkeypatch.setattr(kernels, "_current_device", lambda: -1)
    pool, table, pos = torch.zeros(4, 1, 1, 2, 16, 80, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    rows, far = torch.zeros(2, 128), torch.empty_strided((2, 128), (2 ** 32 + 128, 1), device="meta")
    for layer in (2 ** 32, -2 ** 32, 2 ** 33 + 1, 2 ** 31):
        for call in (lambda: kernels.kv4_append(rows, rows, pool, pos, layer=layer, block_table=table), lambda: kernels.kv4_read(pool, pos, layer=layer, block_table=table)):
            with pytest.raises(ValueError):
                call()
    for call in (lambda: kernels.kv4_append(far, far, pool, pos, layer=0, block_table=table), lambda: kernels.kv4_read(pool, pos, layer=0, block_table=table, k=far, v=far),
                 lambda: kernels.attention_kv4(far, pool, pos, layer=0, n_q=1, block_table=table), lambda: kernels.beam_select(far, torch.zeros(2), beams=2, k=2)):
        with pytest.raises(ValueError):
            call()
    one = torch.zeros(200).as_strided((1, 128), (2 ** 32 + 64, 1))
    assert kernels._arg_rows(one, -1, 128, "k") == (one.data_ptr(), 128, 1)


@pytest.mark.parametrize("shift,code", [(0, -1), (4, -1), (16, -1), (76, -1), (-4, -1), (-76, -1)])
def test_reorder_into_a_part_of_the_table_itself(lib, shift, code):
    """A table of 4 rows of 5 entries is 80 bytes long."""
    c = cache()
    assert lib.tenzo_cuda_kv4_reorder(C.byref(c), P + shift, P, P, 2, 2, 0, None) == code
    for beside in (80, -80):                             # (without a device the launch fails; on one it is not tried)
        assert torch.cuda.is_available() or lib.tenzo_cuda_kv4_reorder(C.byref(c), P + beside, P, P, 2, 2, 0, None) > 0


@pytest.mark.parametrize("n_kv,stride", [(1 << 25, 0), (1 << 25, 128), (3 << 24, -(1 << 31)), ((1 << 25) + 1, 128)])
def test_heads_whose_values_pass_32_bits(lib, n_kv, stride):
    """n_kv * 128 is 2^32 and more: no stride holds that many values."""
    c = cache(n_kv=n_kv)
    assert lib.tenzo_cuda_kv4_append(C.byref(c), 0, P, P, stride, P, P, 1, None, None, 0, 0, None) == abi.ERR_INVALID
    assert lib.tenzo_cuda_kv4_read(C.byref(c), 0, P, P, stride, P, P, 1, 0, None) == abi.ERR_INVALID


@pytest.mark.parametrize("n_q,n_kv", [(4 * 65535 + 1, 1), (65536, 65536), (4 * 65536, 65536)])
def test_splits_of_more_heads_than_the_call_takes(lib, n_q, n_kv):
    assert lib.tenzo_cuda_attention_kv4_splits(1, n_q, n_kv, 80) == 0
    assert lib.tenzo_cuda_attention_kv4(C.byref(attention(n_q=n_q, cache=cache(n_kv=n_kv))), None) == abi.ERR_INVALID
    for q, kv in ((4 * 65535, 1), (65535, 65535), (4 * 65535, 65535), (5 * 52428, 52428)):
        assert lib.tenzo_cuda_attention_kv4_splits(1, q, kv, 80) >= 1
