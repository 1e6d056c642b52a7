"""Results of the calls on trees and bounded caches that have bytes in common with what the call reads, or with each other, are refused wherever the overlap begins. Without a device: refusals
come before any launch, and a call that is not refused ends with the runtime's error instead. (With a device that one would run on addresses that mean nothing: not done there.)"""
import ctypes as C

import pytest
import torch
from tenzo_b200 import abi, load_library

S, N = 4, 7
AT = {n: (i + 1) << 24 for i, n in enumerate(["k", "v", "scale_k", "scale_v", "table", "token", "parent", "chosen", "start", "count", "seq", "weight", "position", "length", "protect_from", "q"])}
OUT = 1 << 40


def cache():
    return abi.Kv8Cache(k=AT["k"], v=AT["v"], scale_k=AT["scale_k"], scale_v=AT["scale_v"], n_blocks=10, n_layers=2, n_kv=3, slots=16, block_table=AT["table"], table_rows=6, table_stride=5)


ROWS = 10 * 2 * 3 * 16
POOLS = {"k": ROWS * 128, "v": ROWS * 128, "scale_k": ROWS * 4, "scale_v": ROWS * 4, "table": 6 * 5 * 4, "weight": ROWS * 4, "position": ROWS * 4}


def accept(**over):
    a = dict(cache=cache(), sequences=S, nodes=N, accepted=OUT, next=OUT + S * 4, path=OUT + 2 * S * 4) | {n: AT[n] for n in ("token", "parent", "chosen", "start", "count", "seq", "weight", "position")}
    return load_library().tenzo_cuda_kv8_accept(C.byref(abi.Kv8AcceptArgs(**(a | over))), None)


def evict(**over):
    a = dict(cache=cache(), sequences=S, keep=8, max_len=80, length_out=OUT) | {n: AT[n] for n in ("length", "seq", "protect_from", "weight", "position")}
    return load_library().tenzo_cuda_kv8_evict(C.byref(abi.Kv8EvictArgs(**(a | over))), None)


def tree(**over):
    a = dict(cache=cache(), q=AT["q"], out=OUT, lse=OUT + S * N * 768 * 4, start=AT["start"], n_q=6, sequences=S, nodes=N, max_len=80)
    return load_library().tenzo_cuda_attention_tree(C.byref(abi.AttentionTreeArgs(**(a | over))), None)


WRITTEN = {"accepted": S * 4, "next": S * 4, "path": S * N * 4}
READ = {"token": S * N * 4, "parent": S * N * 4, "chosen": S * N * 4, "start": S * 4, "count": S * 4, "seq": S * 4} | POOLS


@pytest.mark.parametrize("read", READ)
@pytest.mark.parametrize("written", WRITTEN)
def test_accept(written, read):
    assert accept(**{written: AT[read] + READ[read] - 4}) == abi.ERR_INVALID                     # the last word of what is read
    assert accept(**{written: AT[read] - WRITTEN[written] + 4}) == abi.ERR_INVALID               # the first one


def test_accept_results_apart_from_each_other():
    assert accept(next=OUT + S * 4 - 4) == accept(path=OUT + 2 * S * 4 - 4) == accept(path=OUT - S * N * 4 + 4, next=OUT + 4096) == abi.ERR_INVALID


@pytest.mark.parametrize("read", {"length": S * 4, "seq": S * 4, "protect_from": S * 4} | POOLS)
def test_evict(read):
    size = POOLS.get(read, S * 4)
    assert evict(length_out=AT[read] + size - 4) == evict(length_out=AT[read] - S * 4 + 4) == abi.ERR_INVALID


def test_attention():
    q, out, lse = S * N * 768 * 4, S * N * 768 * 4, S * N * 6 * 4
    assert tree(out=AT["q"] + q - 16) == tree(out=AT["q"] - out + 16) == abi.ERR_INVALID
    assert tree(lse=AT["q"] + q - 4) == tree(lse=AT["q"] - lse + 4) == tree(lse=OUT + out - 4) == tree(lse=OUT - lse + 4) == abi.ERR_INVALID


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses mean nothing")
def test_what_lies_side_by_side_is_not_refused():
    for rc in (accept(), evict(), tree(), evict(length_out=AT["length"] + S * 4), evict(length_out=AT["length"] - S * 4), tree(lse=AT["q"] - S * N * 6 * 4),
               *(accept(**{w: AT[r] + READ[r]}) for w in WRITTEN for r in READ), *(accept(**{w: AT[r] - WRITTEN[w]}) for w in WRITTEN for r in READ)):
        assert rc not in (0, abi.ERR_INVALID, abi.ERR_UNSUPPORTED)
