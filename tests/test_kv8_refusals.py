"""What the calls on trees and bounded caches refuse, without a device: refusals come before any launch. And the packed arguments of the Python calls are
the C structs."""
import ctypes as C

import pytest
import torch
from tenzo_b200 import abi, kernels, load_library

P = 0x10000                                       # a 16-byte aligned address that nothing looks at


@pytest.fixture(scope="module")
def lib():
    return load_library()


def cache(**over):
    c = abi.Kv8Cache(k=P, v=P, scale_k=P, scale_v=P, n_blocks=10, n_layers=2, n_kv=3, slots=16, block_table=P, table_rows=4, table_stride=5)
    for k, v in over.items():
        setattr(c, k, v)
    return c


def tree(**over):
    a = abi.AttentionTreeArgs(q=P, out=P + (1 << 20), lse=P, cache=cache(), start=P, layer=0, n_q=6, sequences=4, nodes=7, max_len=80)
    for k, v in over.items():
        setattr(a, k, v)
    return a


def call(name, cls, c, a):
    if c is None:
        return getattr(load_library(), name)(None, None)
    return getattr(load_library(), name)(C.byref(cls(cache=c, **a)), None)


def append(lib, c, **over):
    return call("tenzo_cuda_kv8_append", abi.Kv8AppendArgs, c, dict(layer=0, k=P, v=P, kv_stride=384, place=P, seq=P, rows=4, weight=P, position=P) | over)


def evict(lib, c, **over):
    return call("tenzo_cuda_kv8_evict", abi.Kv8EvictArgs, c, dict(weight=P, position=P, length=P, seq=P, sequences=4, keep=8, max_len=80, length_out=P + 64) | over)


def accept(lib, c, **over):
    return call("tenzo_cuda_kv8_accept", abi.Kv8AcceptArgs, c, dict(token=P, parent=P, chosen=P, start=P, seq=P, sequences=4, nodes=7, accepted=P + 64, next=P + 128, path=P + 256) | over)


BAD_CACHES = [dict(k=None), dict(v=None), dict(scale_k=None), dict(scale_v=None), dict(k=P + 8), dict(v=P + 4), dict(scale_k=P + 4), dict(scale_v=P + 8), dict(block_table=None),
              dict(n_blocks=0), dict(n_layers=0), dict(n_kv=0), dict(slots=0), dict(slots=8), dict(slots=24), dict(slots=-16), dict(table_rows=0), dict(table_stride=0),
              dict(n_blocks=1 << 20, n_layers=1 << 5, slots=1 << 6), dict(n_blocks=1 << 30, n_layers=1 << 30)]


@pytest.mark.parametrize("over", BAD_CACHES, ids=str)
def test_caches(lib, over):
    c = cache(**over)
    assert append(lib, c) == evict(lib, c) == accept(lib, c) == abi.ERR_INVALID
    a = tree(cache=c)
    assert lib.tenzo_cuda_attention_tree(C.byref(a), None) == lib.tenzo_cuda_kv8_weigh(C.byref(a), P, None) == abi.ERR_INVALID


def test_null(lib):
    assert append(lib, None) == evict(lib, None) == accept(lib, None) == lib.tenzo_cuda_attention_tree(None, None) == lib.tenzo_cuda_kv8_weigh(None, P, None) == abi.ERR_INVALID


@pytest.mark.parametrize("over", [dict(layer=-1), dict(layer=2), dict(k=None), dict(v=None), dict(kv_stride=383), dict(place=None), dict(rows=-1), dict(seq=None, rows=5), dict(rope_cos=P),
                                  dict(rope_sin=P), dict(rope_cos=P, rope_sin=P, rope_len=0), dict(rope_cos=P + 4, rope_sin=P, rope_len=9), dict(rope_cos=P, rope_sin=P + 8, rope_len=9)], ids=str)
def test_append(lib, over):
    assert append(lib, cache(), **over) == abi.ERR_INVALID


TREE = [dict(q=None), dict(start=None), dict(layer=2), dict(layer=-1), dict(n_q=0), dict(n_q=7), dict(n_q=-6), dict(sequences=-1), dict(nodes=0), dict(nodes=-1), dict(max_len=0), dict(max_len=81),
        dict(cache=cache(table_rows=3)), dict(rope_cos=P), dict(rope_sin=P), dict(rope_cos=P, rope_sin=P, rope_len=0), dict(q_stride=767), dict(q_stride=-768), dict(nodes=40, mask=P, mask_stride=1),
        dict(mask=P, mask_stride=-1)]


@pytest.mark.parametrize("over", TREE, ids=str)
def test_tree_and_weigh(lib, over):
    a = tree(**over)
    assert lib.tenzo_cuda_attention_tree(C.byref(a), None) == abi.ERR_INVALID
    assert lib.tenzo_cuda_kv8_weigh(C.byref(a), P, None) == abi.ERR_INVALID


@pytest.mark.parametrize("over", [dict(out=None), dict(out=P + (1 << 20) + 4), dict(out=P), dict(out=P + 27 * 768 * 4), dict(out=P, q=P + 27 * 768 * 4), dict(out=P + (27 * 800 + 764) * 4, q=P, q_stride=800), dict(shares=-1), dict(shares=65536), dict(shares=3), dict(shares=3, workspace=P + 8, workspace_bytes=1 << 30),
                                  dict(shares=3, workspace=P, workspace_bytes=100)], ids=str)
def test_tree_alone(lib, over):
    assert lib.tenzo_cuda_attention_tree(C.byref(tree(**over)), None) == abi.ERR_INVALID


def test_weigh_alone(lib):
    assert lib.tenzo_cuda_kv8_weigh(C.byref(tree()), None, None) == abi.ERR_INVALID
    assert lib.tenzo_cuda_kv8_weigh(C.byref(tree(lse=None)), P, None) == abi.ERR_INVALID


def test_too_many_nodes(lib):
    a = tree(nodes=257)
    assert lib.tenzo_cuda_attention_tree(C.byref(a), None) == lib.tenzo_cuda_kv8_weigh(C.byref(a), P, None) == accept(lib, cache(), nodes=257) == abi.ERR_UNSUPPORTED


def test_workspace(lib):
    need = lib.tenzo_cuda_attention_tree_workspace_bytes
    assert need(0, 4, 4, 2, 0) == need(1, 0, 4, 2, 0) == need(1, 257, 4, 2, 0) == need(1, 4, 0, 2, 0) == need(1, 4, 5, 2, 0) == need(1, 4, 4, 2, -1) == need(1, 4, 4, 2, 65536) == 0
    for sequences, nodes, n_q, n_kv in ((1, 1, 20, 5), (1, 64, 20, 5), (64, 16, 20, 5), (3, 256, 7, 1), (1, 1, 1, 1), (5000, 3, 32, 32), (2, 256, 64, 1)):
        room = need(sequences, nodes, n_q, n_kv, 0)
        assert 0 < room - 8 * sequences * n_kv < 64 << 20 and room == kernels.attention_tree_workspace_bytes(sequences, nodes, n_q, n_kv)
        assert need(sequences, nodes, n_q, n_kv, 7) < need(sequences, nodes, n_q, n_kv, 9)
    assert need(2, 1, 4, 2, 10) == 32 + 10 * 2 * 16 * 520                       # 2 * 2 words, and two sets of sixteen rows a share


@pytest.mark.parametrize("over,code", [(dict(weight=None), -1), (dict(position=None), -1), (dict(weight=P + 4), -1), (dict(position=P + 8), -1), (dict(length=None), -1), (dict(length_out=None), -1), (dict(length_out=P), -1), (dict(length_out=P + 128, seq=P + 128), -1), (dict(length_out=P + 128, protect_from=P + 128), -1), (dict(keep=0), -1), (dict(keep=-3), -1),
                                       (dict(max_len=0), -1), (dict(max_len=81), -1), (dict(sequences=-1), -1), (dict(seq=None, sequences=5), -1), (dict(sequences=65536), -5)], ids=str)
def test_evict(lib, over, code):
    assert evict(lib, cache(), **over) == code


def test_evict_too_long(lib):
    c = cache(table_stride=(1 << 16) + 1)
    assert evict(lib, c, max_len=(1 << 20) + 1) == abi.ERR_UNSUPPORTED


@pytest.mark.parametrize("over,code", [(dict(token=None), -1), (dict(parent=None), -1), (dict(chosen=None), -1), (dict(start=None), -1), (dict(accepted=None), -1), (dict(next=None), -1),
                                       (dict(path=None), -1), (dict(accepted=P), -1), (dict(next=P), -1), (dict(path=P), -1), (dict(count=P + 64), -1), (dict(nodes=0), -1), (dict(sequences=-1), -1), (dict(seq=None, sequences=5), -1), (dict(sequences=65536), -5)], ids=str)
def test_accept(lib, over, code):
    assert accept(lib, cache(), **over) == code


def test_nothing_to_do_is_no_error(lib):
    assert append(lib, cache(), rows=0, k=None, place=None) == 0
    assert evict(lib, cache(), sequences=0, weight=None) == accept(lib, cache(), sequences=0, token=None) == 0
    a = tree(sequences=0, q=None)
    assert lib.tenzo_cuda_attention_tree(C.byref(a), None) == lib.tenzo_cuda_kv8_weigh(C.byref(a), P, None) == 0


def _leaves(cls):
    return [x for _, t in cls._fields_ for x in (_leaves(t) if issubclass(t, C.Structure) else [t])]


def _flat(o):
    return [x for n, t in o._fields_ for x in (_flat(getattr(o, n)) if issubclass(t, C.Structure) else [getattr(o, n)])]


@pytest.mark.parametrize("cls,packer", [(abi.Kv8Cache, kernels._KV8_CACHE), (abi.AttentionTreeArgs, kernels._ATTENTION_TREE), (abi.Kv8AppendArgs, kernels._KV8_APPEND),
                                        (abi.Kv8EvictArgs, kernels._KV8_EVICT), (abi.Kv8AcceptArgs, kernels._KV8_ACCEPT)], ids=lambda x: getattr(x, "__name__", ""))
def test_packed_arguments_are_the_struct(cls, packer):
    values = [1000 + i for i in range(len(_leaves(cls)))]
    assert _flat(cls.from_buffer_copy(packer.pack(*values))) == values


def test_python_calls_refuse_what_is_not_on_the_device():
    c = kernels.Kv8Cache(*(torch.zeros(3, 1, 2, 16, 128, dtype=torch.int8) for _ in range(2)), *(torch.zeros(3, 1, 2, 16) for _ in range(2)), torch.zeros(1, 3, dtype=torch.int32))
    ints = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: kernels.kv8_append(torch.zeros(1, 256), torch.zeros(1, 256), c, ints, layer=0),
                 lambda: kernels.attention_tree(torch.zeros(1, 512), c, ints, layer=0, n_q=4, nodes=1),
                 lambda: kernels.kv8_weigh(torch.zeros(1, 512), torch.zeros(1, 4), c, c.scale_k, ints, layer=0, n_q=4, nodes=1),
                 lambda: kernels.kv8_evict(c, c.scale_k, torch.zeros(3, 1, 2, 16, dtype=torch.int32), ints, keep=4),
                 lambda: kernels.kv8_accept(c, ints[None], ints[None], ints[None], ints)):
        with pytest.raises((ValueError, RuntimeError, AssertionError)):
            call()
