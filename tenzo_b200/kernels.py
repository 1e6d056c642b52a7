"""Per-kernel Python entry points over include/tenzo_kernels.h.

torch is used for device memory and the current stream only; every function is exactly one call
through the C ABI into libtenzo_runtime.so and raises if that call reports an error. There is no
eager/PyTorch fallback.
"""
from __future__ import annotations

import ctypes as C
import functools
import struct
from typing import NamedTuple

import torch

from . import abi, load_library

EPI_STORE, EPI_RESIDUAL, EPI_RELU2_GLU = 0, 1, 2
_TL1_ARGS = struct.Struct("@PPifPii3i3fiPPPPPiiiPNPi0P")       # abi.Tl1GemvArgs
assert _TL1_ARGS.size == C.sizeof(abi.Tl1GemvArgs)


@functools.cache
def _tl1_gemv_packed():
    """tenzo_cuda_tl1_gemv for this module: a prototype of its own, which takes the bytes of _TL1_ARGS and no other object. The
    library's shared one (abi.py) takes an abi.Tl1GemvArgs."""
    fn = load_library()["tenzo_cuda_tl1_gemv"]
    fn.restype, fn.argtypes = C.c_int, [C.c_char_p, C.c_void_p]
    return fn


def _stream() -> int:
    # (0.75 us; torch.cuda.current_stream().cuda_stream gives the same handle by way of a Python object, in 3.3)
    return torch.accelerator.current_stream().native_handle


def _ptr(t: torch.Tensor | None) -> int | None:
    if t is None:
        return None
    assert t.is_cuda and t.is_contiguous()
    return t.data_ptr()


def _rows(t: torch.Tensor | None) -> int | None:
    """Pointer of a 2-D tensor whose rows are contiguous but may be strided (a column slice of a wider buffer)."""
    if t is None:
        return None
    assert t.is_cuda and t.dim() == 2 and t.stride(1) == 1
    return t.data_ptr()


def _ok(rc: int, what: str):
    if rc != 0:
        raise RuntimeError(f"{what} failed: rc={rc}" + (f" ({torch.cuda.get_device_name()})" if rc > 0 else " (bad arguments)"))


def tl1_gemv(x: torch.Tensor, w: torch.Tensor, n_blocks: int, K: int, scales, seg_ends=None, *, epilogue=EPI_STORE,
             resid=None, norm_w=None, do_norm=False, eps=1e-5, want_acc=False, want_act=False, use_pdl=False, out=None, prefetch=None,
             workspace=None):
    """x [batch, K] fp32, w TL1-packed uint8. Returns dict(out=..., acc=..., a=..., inv=...)."""
    lib = load_library()
    batch = x.shape[0]
    n_out = n_blocks * 64 // (2 if epilogue == EPI_RELU2_GLU else 1)
    if out is None:
        out = torch.empty(batch, n_out, dtype=torch.float32, device=x.device)
    acc = torch.empty(batch, n_blocks * 64, dtype=torch.int32, device=x.device) if want_acc else None
    a8 = torch.empty(batch, K, dtype=torch.int8, device=x.device) if want_act else None
    inv = torch.empty(batch, dtype=torch.float32, device=x.device) if want_act else None
    scales = (*scales, 0.0, 0.0, 0.0)[:max(3, len(scales))]
    seg_ends = (n_blocks,) * 3 if seg_ends is None else (*seg_ends, n_blocks, n_blocks, n_blocks)[:max(3, len(seg_ends))]
    ws = workspace
    if batch > 1 and ws is None:
        ws = torch.empty(lib.tenzo_cuda_tl1_gemv_workspace_bytes(batch, K), dtype=torch.uint8, device=x.device)
    # Packed in one go: a one-sequence call is bound by this function, not by its kernel (22 attribute assignments take 2.2 us).
    g = _TL1_ARGS.pack(_ptr(x), _ptr(norm_w) or 0, do_norm, eps, _ptr(w) or 0, n_blocks, K, *seg_ends, *scales, epilogue, _ptr(resid) or 0, _ptr(out),
                       _ptr(acc) or 0, _ptr(a8) or 0, _ptr(inv) or 0, batch, x.stride(0), out.stride(0), _ptr(prefetch) or 0,
                       0 if prefetch is None else prefetch.numel() * prefetch.element_size(), _ptr(ws) or 0, use_pdl)
    _ok(_tl1_gemv_packed()(g, _stream()), "tenzo_cuda_tl1_gemv")
    return dict(out=out, acc=acc, a=a8, inv=inv)


def rmsnorm_quant(x: torch.Tensor, norm_w=None, *, do_norm=True, eps=1e-5, qmax=31, want_y=True, want_q=True):
    lib = load_library()
    batch, dim = x.shape
    y = torch.empty_like(x) if want_y else None
    q = torch.empty(batch, dim, dtype=torch.int8, device=x.device) if want_q else None
    s = torch.empty(batch, dtype=torch.float32, device=x.device) if want_q else None
    _ok(lib.tenzo_cuda_rmsnorm_quant(_ptr(x), _ptr(norm_w), int(do_norm), eps, dim, qmax, batch, x.stride(0), _ptr(y),
                                     _ptr(q), _ptr(s), _stream()), "tenzo_cuda_rmsnorm_quant")
    return y, q, s


def attention_workspace_bytes(batch, n_q, n_kv, max_len) -> int:
    return int(load_library().tenzo_cuda_attention_workspace_bytes(batch, n_q, n_kv, max_len))


def attention_int8(q, k, v, cache_k, cache_v, scale_k, scale_v, pos, *, layer, n_q, n_kv, max_seq, rope_cos=None,
                   rope_sin=None, append=True, max_len=None, use_pdl=False, heads_per_cta=0, out=None, tiles=0,
                   block_table=None, n_layers=0, mode=0, split_keys=0, workspace=None):
    """q [batch, n_q*128], k/v [batch, n_kv*128]; caches [batch, layers, n_kv, max_seq, 128] int8 and
    [batch, layers, n_kv, max_seq] fp32; pos int32 [batch]. Returns out [batch, n_q*128].
    With block_table (int32 [batch, blocks per sequence]) the caches are the paged_int8 pools
    [blocks, n_layers, n_kv, 16, 128] / [blocks, n_layers, n_kv, 16] and the arithmetic is the paged cache's."""
    lib = load_library()
    batch = q.shape[0]
    if max_len is None:
        max_len = int(pos.max().item()) + 1
    if out is None:
        out = torch.empty(batch, n_q * 128, dtype=torch.float32, device=q.device)
    a = abi.AttentionArgs()
    a.q, a.k, a.v, a.out = _rows(q), _rows(k), _rows(v), _ptr(out)
    a.q_stride, a.kv_stride = q.stride(0), (k.stride(0) if k is not None else 0)
    a.cache_k, a.cache_v, a.scale_k, a.scale_v = _ptr(cache_k), _ptr(cache_v), _ptr(scale_k), _ptr(scale_v)
    a.seq_stride_kv, a.seq_stride_sc = cache_k.stride(0), scale_k.stride(0)
    a.pos, a.rope_cos, a.rope_sin = _ptr(pos), _ptr(rope_cos), _ptr(rope_sin)
    a.layer, a.n_q, a.n_kv, a.head_dim, a.max_seq = layer, n_q, n_kv, 128, max_seq
    a.batch, a.max_len, a.append, a.use_pdl, a.heads_per_cta = batch, max_len, int(append), int(use_pdl), heads_per_cta
    a.tiles = tiles
    if block_table is not None:
        assert block_table.dtype == torch.int32 and block_table.is_contiguous()
        a.block_table, a.table_stride, a.n_layers = _ptr(block_table), (block_table.stride(0) if block_table.dim() == 2 else 0), n_layers
        a.n_pool_blocks = cache_k.shape[0]
    if workspace is None and (mode == 1 or tiles in (0, 3)):
        need = lib.tenzo_cuda_attention_workspace_bytes if mode == 1 else lib.tenzo_cuda_attention_exact_workspace_bytes
        workspace = torch.empty(need(batch, n_q, n_kv, max_len), dtype=torch.uint8, device=q.device)
    if workspace is not None:
        a.workspace, a.workspace_bytes = _ptr(workspace), workspace.numel()
    a.mode, a.split_keys = mode, split_keys
    _ok(lib.tenzo_cuda_attention_int8(C.byref(a), _stream()), "tenzo_cuda_attention_int8")
    return out


def lm_head_i8(x, w, row_scales, *, norm_w=None, do_norm=True, eps=1e-5, want_logits=True, want_acc=False, use_pdl=False, logits=None):
    lib = load_library()
    batch, hidden = x.shape
    vocab = w.shape[0]
    if logits is None and want_logits:
        logits = torch.empty(batch, vocab, dtype=torch.float32, device=x.device)
    acc = torch.empty(batch, vocab, dtype=torch.int32, device=x.device) if want_acc else None
    arg = torch.empty(batch, dtype=torch.int32, device=x.device)
    scratch = torch.empty(lib.tenzo_cuda_lm_head_scratch_bytes(batch), dtype=torch.uint8, device=x.device)
    _ok(lib.tenzo_cuda_lm_head_i8(_ptr(x), _ptr(norm_w), int(do_norm), eps, _ptr(w), _ptr(row_scales), vocab, hidden,
                                  batch, x.stride(0), _ptr(logits), _ptr(acc), _ptr(arg), _ptr(scratch), int(use_pdl),
                                  _stream()), "tenzo_cuda_lm_head_i8")
    return logits, acc, arg


def lm_head_i8_static(x, w, row_scales, *, norm_w=None, do_norm=True, eps=1e-5, logits=None, argmax=None, use_pdl=False):
    """LM head through the allocation-free entry point: the caller passes every buffer (logits
    [batch, vocab] fp32 and argmax [batch] int32, both preallocated); the library allocates nothing."""
    lib = load_library()
    batch, hidden = x.shape
    _ok(lib.tenzo_cuda_lm_head_i8_static(_ptr(x), _ptr(norm_w), int(do_norm), eps, _ptr(w), _ptr(row_scales), w.shape[0],
                                         hidden, batch, x.stride(0), _ptr(logits), None, _ptr(argmax), int(use_pdl), _stream()),
        "tenzo_cuda_lm_head_i8_static")
    return logits, argmax


def embedding_i8(w, row_scales, tokens):
    lib = load_library()
    batch, hidden = tokens.shape[0], w.shape[1]
    x = torch.empty(batch, hidden, dtype=torch.float32, device=w.device)
    _ok(lib.tenzo_cuda_embedding_i8(_ptr(w), _ptr(row_scales), hidden, _ptr(tokens), batch, _ptr(x), hidden, w.shape[0], _stream()),
        "tenzo_cuda_embedding_i8")
    return x


def tl1_pack_rows2bit(raw, N, K):
    lib = load_library()
    packed = torch.empty(N * K // 4, dtype=torch.uint8, device=raw.device)
    _ok(lib.tenzo_cuda_tl1_pack_rows2bit(_ptr(raw), N, K, _ptr(packed), _stream()), "tenzo_cuda_tl1_pack_rows2bit")
    return packed


# ---- 4-bit paged cache and beam search -------------------------------------------------------------------------------------------
_KV4_CACHE = struct.Struct("@PiiiPii0P")                        # abi.Kv4Cache
_KV4_ATTENTION = struct.Struct("@PPPiiiPii0PPPPPiiiiiiiiPN")    # abi.AttentionKv4Args
_BEAM_SELECT = struct.Struct("@PPPiiiiiiiPPPPN")                # abi.BeamSelectArgs
assert _KV4_CACHE.size == C.sizeof(abi.Kv4Cache) and _KV4_ATTENTION.size == C.sizeof(abi.AttentionKv4Args) and _BEAM_SELECT.size == C.sizeof(abi.BeamSelectArgs)


_PI, _PP, _PB = C.c_int, C.c_void_p, C.c_char_p
_INT_MOST = 2 ** 31 - 1


@functools.cache
def _beam_calls():
    """The entry points with prototypes of this module's own, whose structs are the bytes of a struct.Struct; tenzo_cuda_kv4_append, _read, _reorder,
    tenzo_cuda_attention_kv4, tenzo_cuda_beam_select, the two workspace sizes, and the attention's choice of splits."""
    def fn(name, *argtypes, restype=C.c_int):
        f = load_library()[name]
        f.restype, f.argtypes = restype, list(argtypes)
        return f
    return (fn("tenzo_cuda_kv4_append", _PB, _PI, _PP, _PP, _PI, _PP, _PP, _PI, _PP, _PP, _PI, _PI, _PP),
            fn("tenzo_cuda_kv4_read", _PB, _PI, _PP, _PP, _PI, _PP, _PP, _PI, _PI, _PP),
            fn("tenzo_cuda_kv4_reorder", _PB, _PP, _PP, _PP, _PI, _PI, _PI, _PP),
            fn("tenzo_cuda_attention_kv4", _PB, _PP), fn("tenzo_cuda_beam_select", _PB, _PP),
            fn("tenzo_cuda_attention_kv4_workspace_bytes", _PI, _PI, _PI, _PI, restype=C.c_size_t),
            fn("tenzo_cuda_beam_select_workspace_bytes", _PI, _PI, _PI, _PI, restype=C.c_size_t), fn("tenzo_cuda_attention_kv4_splits", _PI, _PI, _PI, _PI))


# (These calls take as long as their kernels at small sizes: attributes of a tensor are read once, 0.05 us each, and the stream's handle comes from
# the raw getter, 0.07 us against 0.76 by way of a stream object.)
_current_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _refuse(t, what, need):
    raise ValueError(f"{what}: {need} on the current CUDA device is needed, not {t.dtype} {tuple(t.shape)} of strides {t.stride()} on {t.device}")


def _arg(t: torch.Tensor | None, dtype, device: int, what: str) -> int:
    """Address of a contiguous tensor of `dtype` on `device`; 0 for None."""
    if t is None:
        return 0
    if t.dtype is not dtype or t.get_device() != device or not t.is_contiguous():
        _refuse(t, what, f"a contiguous {dtype} tensor")
    return t.data_ptr()


def _arg_rows(t: torch.Tensor, device: int, columns: int, what: str) -> tuple[int, int, int]:
    """Address, row stride and number of fp32 rows that may lie apart (a column slice of a wider buffer)."""
    shape, strides = t.shape, t.stride()
    n = shape[0] if len(shape) == 2 else -1
    if n < 0 or t.dtype is not torch.float32 or t.get_device() != device or shape[1] != columns or (columns > 1 and strides[1] != 1) or (n > 1 and strides[0] < columns):
        _refuse(t, what, f"fp32 rows of {columns} values that do not overlap")
    stride = strides[0] if n > 1 else max(strides[0], columns)
    if stride > _INT_MOST:
        if n > 1:
            _refuse(t, what, "rows that lie fewer than 2^31 values apart")
        stride = columns                                        # one row: any
    return t.data_ptr(), stride, n


def _kv4_cache(pool: torch.Tensor, block_table: torch.Tensor, device: int):
    """The fields of abi.Kv4Cache."""
    shape, table = pool.shape, block_table.shape
    if len(shape) != 6 or len(table) != 2 or shape[3] != 2 or shape[4] != 16 or shape[5] != 80:
        raise ValueError(f"a pool [blocks, layers, kv heads, 2, 16, 80] and a table [rows, columns] are needed, not {tuple(shape)} and {tuple(table)}")
    return _arg(pool, torch.uint8, device, "pool"), shape[0], shape[1], shape[2], _arg(block_table, torch.int32, device, "block_table"), table[0], table[1]


def _arg_layer(layer: int) -> int:
    """`layer` where it fits the prototype's C int, which takes larger ones modulo 2^32."""
    if not -_INT_MOST <= layer <= _INT_MOST:
        raise ValueError(f"there is no layer {layer}")
    return layer


def _arg_entries(t, n: int, device: int, what: str) -> int:
    """Address of int32 [n]; 0 for None."""
    if t is not None and t.shape != (n,):
        raise ValueError(f"{what} has one entry for each of {n} rows, not {tuple(t.shape)}")
    return _arg(t, torch.int32, device, what)


def _arg_rope(cos, sin, device: int) -> tuple[int, int, int]:
    if cos is None and sin is None:
        return 0, 0, 0
    shape = None if cos is None or sin is None else cos.shape
    if shape is None or len(shape) != 2 or shape[1] != 64 or sin.shape != shape:
        raise ValueError("rope_cos and rope_sin are tables of the same number of rows of 64")
    return _arg(cos, torch.float32, device, "rope_cos"), _arg(sin, torch.float32, device, "rope_sin"), shape[0]


def kv4_append(k, v, pool, pos, *, layer, block_table, seq=None, rope_cos=None, rope_sin=None, use_pdl=False):
    """Rotates the rows k [n, n_kv*128], quantises k and v to 4 bits and stores them in `pool` (uint8 [blocks, layers, n_kv, 2, 16, 80]) at
    positions pos int32 [n] of the sequences seq int32 [n] (default: row i is sequence i) of block_table int32 [sequences, columns].
    A negative position marks a padding row, for which nothing is stored."""
    dev = _current_device()
    cache = _kv4_cache(pool, block_table, dev)
    n_kv = cache[3]
    (kp, ks, n), (vp, vs, m) = _arg_rows(k, dev, n_kv * 128, "k"), _arg_rows(v, dev, n_kv * 128, "v")
    if n != m or (ks != vs and n > 1):
        raise ValueError("k and v have the same number of rows, equally far apart")
    cos, sin, length = _arg_rope(rope_cos, rope_sin, dev)
    _ok(_beam_calls()[0](_KV4_CACHE.pack(*cache), _arg_layer(layer), kp, vp, ks, _arg_entries(pos, n, dev, "pos"), _arg_entries(seq, n, dev, "seq"), n, cos, sin, length, use_pdl, _raw_stream(dev)),
        "tenzo_cuda_kv4_append")


def kv4_read(pool, pos, *, layer, block_table, seq=None, use_pdl=False, k=None, v=None):
    """The rows at positions pos int32 [n] of the sequences seq as the cache holds them: (k, v), fp32 [n, n_kv*128], the keys rotated; zeros for
    negative positions. k and v may be given (both) to be written into."""
    dev, n = _current_device(), len(pos)
    cache = _kv4_cache(pool, block_table, dev)
    ks = cache[3] * 128
    if k is None and v is None:
        both = torch.empty(2, n, ks, dtype=torch.float32, device=pool.device)
        kp = both.data_ptr()
        vp = kp + 4 * n * ks
        k, v = both.unbind(0)
    elif k is None or v is None:
        raise ValueError("k and v are given both or not at all")
    else:
        (kp, ks, m), (vp, vs, o) = _arg_rows(k, dev, ks, "k"), _arg_rows(v, dev, ks, "v")
        if n != m or n != o or (ks != vs and n > 1):
            raise ValueError("k and v have one row for each position, equally far apart")
    _ok(_beam_calls()[1](_KV4_CACHE.pack(*cache), _arg_layer(layer), kp, vp, ks, _arg_entries(pos, n, dev, "pos"), _arg_entries(seq, n, dev, "seq"), n, use_pdl, _raw_stream(dev)), "tenzo_cuda_kv4_read")
    return k, v


@functools.lru_cache(1024)
def attention_kv4_workspace_bytes(rows, n_q, n_kv, max_len) -> int:
    """Enough for any split_keys."""
    return _beam_calls()[5](rows, n_q, n_kv, max_len)


@functools.lru_cache(1024)
def _attention_kv4_room(rows, n_q, n_kv, max_len, split_keys) -> int:
    """What one call needs: splits of split_keys keys, or as many as it chooses itself."""
    splits = -(-max_len // (-(-split_keys // 128) * 128)) if split_keys > 0 else _beam_calls()[7](rows, n_q, n_kv, max_len)
    return rows * n_q * 520 * splits if splits > 1 else 0


@functools.lru_cache(1024)
def beam_select_workspace_bytes(groups, beams, vocab, k) -> int:
    return _beam_calls()[6](groups, beams, vocab, k)


def attention_kv4(q, pool, pos, *, layer, n_q, block_table, seq=None, rope_cos=None, rope_sin=None, max_len=None, split_keys=0, use_pdl=False, out=None,
                  workspace=None):
    """GQA attention of the query rows q [rows, n_q*128] over the keys 0 .. pos[row] of their sequences in the 4-bit pool, the queries rotated first.
    Returns out [rows, n_q*128]; zeros where pos is negative. max_len: an upper bound on pos + 1 (default: what the table has room for).
    workspace: a uint8 tensor for partial results of splits (default: one is allocated if the call wants it)."""
    dev = _current_device()
    cache = _kv4_cache(pool, block_table, dev)
    n_kv, columns = cache[3], cache[6]
    qp, q_stride, rows = _arg_rows(q, dev, n_q * 128, "q")
    cos, sin, length = _arg_rope(rope_cos, rope_sin, dev)
    if max_len is None:
        max_len = min(columns * 16, length) if cos else columns * 16
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != (rows, n_q * 128):
        raise ValueError(f"out is [{rows}, {n_q * 128}]")
    if workspace is None:
        size = _attention_kv4_room(rows, n_q, n_kv, max_len, split_keys)
        if size:
            workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
    args = _KV4_ATTENTION.pack(qp, _arg(out, torch.float32, dev, "out"), *cache, _arg_entries(pos, rows, dev, "pos"), _arg_entries(seq, rows, dev, "seq"),
                               cos, sin, length, q_stride, layer, n_q, rows, max_len, split_keys, use_pdl, _arg(workspace, torch.uint8, dev, "workspace"),
                               0 if workspace is None else workspace.numel())
    _ok(_beam_calls()[3](args, _raw_stream(dev)), "tenzo_cuda_attention_kv4")
    return out


def beam_select(logits, scores, *, beams, k, finished=None, eos=0, use_pdl=False, workspace=None):
    """The k best continuations of each group of `beams` rows of logits [groups*beams, vocab], given the beams' sums of log-probabilities scores
    fp32 [groups*beams]. Returns (parent, token, score), [groups, k], best first. finished int32 [groups*beams]: beams that only go on with `eos`."""
    dev, vocab = _current_device(), logits.shape[-1]
    lp, stride, rows = _arg_rows(logits, dev, vocab, "logits")
    groups = rows // beams if beams > 0 else -1
    if k < 1 or groups * beams != rows or scores.shape != (rows,):
        raise ValueError(f"{rows} rows of logits are no groups of {beams} beams with one score each, or k = {k} is no number of candidates")
    device = logits.device
    parent, token, score = torch.empty(3, groups, k, dtype=torch.int32, device=device).unbind(0)
    score = score.view(torch.float32)
    if workspace is None:
        workspace = torch.empty(beam_select_workspace_bytes(groups, beams, vocab, k), dtype=torch.uint8, device=device)
    args = _BEAM_SELECT.pack(lp, _arg(scores, torch.float32, dev, "scores"), _arg_entries(finished, rows, dev, "finished"), eos, stride, groups, beams, vocab, k,
                             use_pdl, parent.data_ptr(), token.data_ptr(), score.data_ptr(), _arg(workspace, torch.uint8, dev, "workspace"), workspace.numel())
    _ok(_beam_calls()[4](args, _raw_stream(dev)), "tenzo_cuda_beam_select")
    return parent, token, score


def kv4_reorder(pool, block_table, parent, length, *, out=None, use_pdl=False):
    """The block table of the beams that go on from parent int32 [groups, beams] of beams that hold length int32 [groups] tokens each. Full blocks are
    shared; the block being filled is copied within `pool` for the second and further children of a beam, into those of beams without children."""
    dev, (groups, beams) = _current_device(), parent.shape
    cache = _kv4_cache(pool, block_table, dev)
    rows = cache[5]
    if rows != groups * beams:
        raise ValueError(f"{groups} groups of {beams} beams need as many table rows, not {rows}")
    if out is None:
        out = torch.empty_like(block_table)
    elif out.shape != block_table.shape:
        raise ValueError("out has the table's shape")
    _ok(_beam_calls()[2](_KV4_CACHE.pack(*cache), _arg(out, torch.int32, dev, "out"), _arg(parent, torch.int32, dev, "parent"), _arg_entries(length, groups, dev, "length"), groups, beams,
                         use_pdl, _raw_stream(dev)), "tenzo_cuda_kv4_reorder")
    return out


def kv4_take_errors() -> int:
    """Error flags of the 4-bit cache's kernels since the last call (1: a wait was given up, 2: an index out of range), -1 if the query failed; waits for
    all streams of the device."""
    return int(load_library().tenzo_cuda_kv4_take_errors())


# ---- INT8 caches: drafted trees, and caches of a bounded number of tokens ------------------------------------------------------------
class Kv8Cache(NamedTuple):
    """The INT8 caches of attention_int8 behind a block table: k, v int8 [blocks, layers, n_kv, slots, 128], scale_k, scale_v fp32 [blocks, layers, n_kv, slots],
    block_table int32 [sequences, columns]; the token at place t of a sequence lies in block block_table[sequence, t / slots], slot t % slots. The paged_int8 pools
    have 16 slots; the contiguous caches are blocks of max_seq slots (a multiple of 16) behind a table of one column, arange(sequences)."""
    k: torch.Tensor
    v: torch.Tensor
    scale_k: torch.Tensor
    scale_v: torch.Tensor
    block_table: torch.Tensor


_KV8_CACHE = struct.Struct("@PPPPiiiiPii0P")                            # abi.Kv8Cache
_ATTENTION_TREE = struct.Struct("@PPPPPPPiiiiPii0PPPPPPPPiiiiiiiiiiPN")    # abi.AttentionTreeArgs
_F32, _I32, _I8, _U8 = torch.float32, torch.int32, torch.int8, torch.uint8
_TREE_WHOLE = 512                                                      # max_len to which the attention cuts no sequence, and needs no workspace
_KV8_APPEND = struct.Struct("@PPPPiiiiPiiPPPPPPPPPiiiii0P")            # abi.Kv8AppendArgs
_KV8_EVICT = struct.Struct("@PPPPiiiiPiiPPPPPPiiii0P")                # abi.Kv8EvictArgs
_KV8_ACCEPT = struct.Struct("@PPPPiiiiPiiPPPPPPPPPPPiii0P")            # abi.Kv8AcceptArgs
for _packer, _struct in ((_KV8_CACHE, abi.Kv8Cache), (_ATTENTION_TREE, abi.AttentionTreeArgs), (_KV8_APPEND, abi.Kv8AppendArgs), (_KV8_EVICT, abi.Kv8EvictArgs), (_KV8_ACCEPT, abi.Kv8AcceptArgs)):
    assert _packer.size == C.sizeof(_struct)


@functools.cache
def _tree_calls():
    """tenzo_cuda_kv8_append, _evict, _accept, tenzo_cuda_attention_tree, tenzo_cuda_kv8_weigh and the attention's workspace, with prototypes of this module's own, whose structs
    are the bytes of a struct.Struct."""
    def fn(name, *argtypes, restype=C.c_int):
        f = load_library()[name]
        f.restype, f.argtypes = restype, list(argtypes)
        return f
    return (fn("tenzo_cuda_kv8_append", _PB, _PP), fn("tenzo_cuda_kv8_evict", _PB, _PP), fn("tenzo_cuda_kv8_accept", _PB, _PP),
            fn("tenzo_cuda_attention_tree", _PB, _PP), fn("tenzo_cuda_kv8_weigh", _PB, _PP, _PP),
            fn("tenzo_cuda_attention_tree_workspace_bytes", _PI, _PI, _PI, _PI, _PI, restype=C.c_size_t))


def _kv8_cache(cache: Kv8Cache, device: int):
    """The fields of abi.Kv8Cache, and the shape of the scales."""
    k, v, sk, sv, table = cache
    shape, rows = k.shape, table.shape
    if len(shape) == 5 and len(rows) == 2:
        blocks, layers, n_kv, slots, dims = shape
        scales = (blocks, layers, n_kv, slots)
        if dims == 128 and v.shape == shape and sk.shape == scales and sv.shape == scales:
            return (_arg(k, _I8, device, "k"), _arg(v, _I8, device, "v"), _arg(sk, _F32, device, "scale_k"), _arg(sv, _F32, device, "scale_v"),
                    blocks, layers, n_kv, slots, _arg(table, _I32, device, "block_table"), *rows), scales
    raise ValueError(f"caches [blocks, layers, kv heads, slots, 128], their scales and a table [rows, columns] are needed, not {tuple(shape)}, {tuple(v.shape)}, "
                     f"{tuple(sk.shape)}, {tuple(sv.shape)} and {tuple(rows)}")


def _arg_beside(t, scales: tuple, dtype, device: int, what: str) -> int:
    """Address of what lies beside the scales; 0 for None."""
    if t is None:
        return 0
    if t.shape != scales:
        raise ValueError(f"{what} has the scales' shape {scales}, not {tuple(t.shape)}")
    return _arg(t, dtype, device, what)


def _arg_int(value: int, what: str) -> int:
    """`value` where it fits the prototype's C int, which takes larger ones modulo 2^32."""
    if not -_INT_MOST <= value <= _INT_MOST:
        raise ValueError(f"{what} is {value}")
    return value


def kv8_append(k, v, cache, place, *, layer, seq=None, rope_pos=None, rope_cos=None, rope_sin=None, weight=None, position=None, use_pdl=False):
    """Rotates the rows k [n, n_kv*128] at rope_pos int32 [n] (default: place), quantises k and v to int8, and stores them at places place int32 [n] of the
    sequences seq int32 [n] (default: row i is sequence i). A scale is max|x| * (1/127), where attention_int8 divides by 127: scales may differ from its own in the last bit, and a code next to a
    border by one. A negative place marks a padding row, for which nothing is stored. weight fp32 and position int32, of the scales' shape, receive 0 and the rotary position."""
    dev = _current_device()
    fields, scales = _kv8_cache(cache, dev)
    n_kv = fields[6]
    (kp, ks, n), (vp, vs, m) = _arg_rows(k, dev, n_kv * 128, "k"), _arg_rows(v, dev, n_kv * 128, "v")
    if n != m or (ks != vs and n > 1):
        raise ValueError("k and v have the same number of rows, equally far apart")
    cos, sin, length = _arg_rope(rope_cos, rope_sin, dev)
    args = _KV8_APPEND.pack(*fields, kp, vp, _arg_entries(place, n, dev, "place"), _arg_entries(seq, n, dev, "seq"), _arg_entries(rope_pos, n, dev, "rope_pos"), cos, sin,
                            _arg_beside(weight, scales, _F32, dev, "weight"), _arg_beside(position, scales, _I32, dev, "position"), _arg_layer(layer), ks, n, length, use_pdl)
    _ok(_tree_calls()[0](args, _raw_stream(dev)), "tenzo_cuda_kv8_append")


@functools.lru_cache(1024)
def attention_tree_workspace_bytes(sequences, nodes, n_q, n_kv, shares=0) -> int:
    return _tree_calls()[5](sequences, nodes, n_q, n_kv, shares)


def _tree_fields(q, cache, start, layer, n_q, nodes, count, mask, seq, rope_pos, rope_cos, rope_sin, max_len, dev):
    """The fields of abi.AttentionTreeArgs from cache to max_len, and what the calls ask further: the query's address, the numbers of rows and sequences, and the scales' shape."""
    fields, scales = _kv8_cache(cache, dev)
    qp, q_stride, rows = _arg_rows(q, dev, n_q * 128, "q")
    sequences = rows // nodes if nodes > 0 else -1
    if sequences * nodes != rows:
        raise ValueError(f"{rows} rows of q are no trees of {nodes} nodes")
    mask_stride = 0
    if mask is not None:
        shape = mask.shape
        if len(shape) != 2 or shape[0] != rows or shape[1] * 32 < nodes:
            raise ValueError(f"mask has a row of at least {-(-nodes // 32)} words for each of {rows} nodes, not {tuple(shape)}")
        mask_stride = shape[1]
    cos, sin, length = _arg_rope(rope_cos, rope_sin, dev)
    if max_len is None:
        max_len = min(fields[7] * fields[10], _INT_MOST)
    return qp, rows, sequences, scales, (*fields, _arg_entries(start, sequences, dev, "start"), _arg_entries(count, sequences, dev, "count"), _arg_entries(seq, sequences, dev, "seq"),
                                 _arg(mask, _I32, dev, "mask"), _arg_entries(rope_pos, rows, dev, "rope_pos"), cos, sin, length, q_stride, mask_stride,
                                 _arg_layer(layer), n_q, sequences, nodes, _arg_int(max_len, "max_len"))


def attention_tree(q, cache, start, *, layer, n_q, nodes, count=None, mask=None, seq=None, rope_pos=None, rope_cos=None, rope_sin=None, max_len=None, want_lse=False,
                   shares=0, use_pdl=False, out=None, lse=None, workspace=None):
    """Attention of the nodes of trees: q [sequences*nodes, n_q*128] over the tokens at places 0 .. start[s] - 1 of sequence s and, of the tree's own at start[s] + j, those
    whose bit j % 32 of mask[row, j / 32] is set (int32 [rows, words]; default: nodes 0 .. i, a chain). start, count int32 [sequences]: tokens that are cached, and nodes
    that are there (default: all); rope_pos int32 [rows]: the queries' rotary positions (default: start + i). Returns out [rows, n_q*128], zeros where nothing is seen;
    with want_lse (out, lse [rows, n_q])."""
    dev = _current_device()
    qp, rows, sequences, _, fields = _tree_fields(q, cache, start, layer, n_q, nodes, count, mask, seq, rope_pos, rope_cos, rope_sin, max_len, dev)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        op = out.data_ptr()
    elif out.shape != (rows, n_q * 128):
        raise ValueError(f"out is [{rows}, {n_q * 128}]")
    else:
        op = _arg(out, _F32, dev, "out")
    lp = 0
    if lse is not None:
        if lse.shape != (rows, n_q):
            raise ValueError(f"lse is [{rows}, {n_q}]")
        lp = _arg(lse, _F32, dev, "lse")
    elif want_lse:
        lse = q.new_empty(rows, n_q)
        lp = lse.data_ptr()
    if workspace is None and shares == 0 and fields[-1] <= _TREE_WHOLE:
        wp = size = 0
    elif workspace is None:
        size = attention_tree_workspace_bytes(sequences, nodes, n_q, fields[6], shares)
        workspace = q.new_empty(-(-size // 4))
        wp = workspace.data_ptr()
    else:
        wp, size = _arg(workspace, _U8, dev, "workspace"), workspace.numel()
    args = _ATTENTION_TREE.pack(qp, op, lp, *fields, _arg_int(shares, "shares"), use_pdl, wp, size)
    _ok(_tree_calls()[3](args, _raw_stream(dev)), "tenzo_cuda_attention_tree")
    return out if lse is None else (out, lse)


def kv8_weigh(q, lse, cache, weight, start, *, layer, n_q, nodes, count=None, mask=None, seq=None, rope_pos=None, rope_cos=None, rope_sin=None, max_len=None, use_pdl=False):
    """Adds to weight (fp32, of the scales' shape) what each cached token received in attention_tree of the same arguments, whose lse [rows, n_q] this reads: the sum of
    softmax's results over the nodes and the query heads of a kv head. Nodes that are refused later count like others; to leave them out, call it behind kv8_accept for the accepted ones,
    which are a chain there: q, lse and rope_pos gathered by its path (anything where that is -1), count=accepted, no mask, the same start."""
    dev = _current_device()
    qp, rows, _, scales, fields = _tree_fields(q, cache, start, layer, n_q, nodes, count, mask, seq, rope_pos, rope_cos, rope_sin, max_len, dev)
    if lse.shape != (rows, n_q):
        raise ValueError(f"lse is [{rows}, {n_q}], not {tuple(lse.shape)}")
    args = _ATTENTION_TREE.pack(qp, 0, _arg(lse, _F32, dev, "lse"), *fields, 0, use_pdl, 0, 0)
    _ok(_tree_calls()[4](args, _arg_beside(weight, scales, _F32, dev, "weight"), _raw_stream(dev)), "tenzo_cuda_kv8_weigh")


def kv8_evict(cache, weight, position, length, *, keep, protect_from=None, seq=None, max_len=None, use_pdl=False):
    """Cuts the sequences that hold length int32 [sequences] tokens back to `keep`, in all layers and for each kv head on its own: the tokens of least weight go, but
    none whose position is protect_from[s] int32 [sequences] or more; those behind place keep - 1 that stay move to the places that became free. Returns the new lengths."""
    dev, sequences = _current_device(), len(length)
    fields, scales = _kv8_cache(cache, dev)
    if max_len is None:
        max_len = min(fields[7] * fields[10], 1 << 20)
    out = torch.empty_like(length)
    args = _KV8_EVICT.pack(*fields, _arg_beside(weight, scales, _F32, dev, "weight"), _arg_beside(position, scales, _I32, dev, "position"),
                           _arg_entries(length, sequences, dev, "length"), _arg_entries(seq, sequences, dev, "seq"), _arg_entries(protect_from, sequences, dev, "protect_from"),
                           out.data_ptr(), sequences, _arg_int(keep, "keep"), _arg_int(max_len, "max_len"), use_pdl)
    _ok(_tree_calls()[1](args, _raw_stream(dev)), "tenzo_cuda_kv8_evict")
    return out


def kv8_accept(cache, token, parent, chosen, start, *, count=None, seq=None, weight=None, position=None, use_pdl=False):
    """The nodes of drafted trees that the model agrees with, given the nodes' tokens, the nodes they go on from and the model's choice after each, int32
    [sequences, nodes] (node 0 is the root); their rows are moved up behind the start[s] cached tokens in all layers. Returns (accepted [sequences], next [sequences],
    path [sequences, nodes]): how many nodes, the root among them, the token chosen after the last, and which nodes, then -1."""
    dev, shape = _current_device(), token.shape
    if len(shape) != 2 or parent.shape != shape or chosen.shape != shape:
        raise ValueError(f"token, parent and chosen are [sequences, nodes], not {tuple(shape)}, {tuple(parent.shape)} and {tuple(chosen.shape)}")
    sequences, nodes = shape
    fields, scales = _kv8_cache(cache, dev)
    tokens = _arg(token, _I32, dev, "token")
    accepted, following, path = token.new_empty(sequences), token.new_empty(sequences), torch.empty_like(token)
    args = _KV8_ACCEPT.pack(*fields, tokens, _arg(parent, _I32, dev, "parent"), _arg(chosen, _I32, dev, "chosen"), _arg_entries(start, sequences, dev, "start"),
                            _arg_entries(count, sequences, dev, "count"), _arg_entries(seq, sequences, dev, "seq"), accepted.data_ptr(), following.data_ptr(), path.data_ptr(),
                            _arg_beside(weight, scales, _F32, dev, "weight"), _arg_beside(position, scales, _I32, dev, "position"), sequences, nodes, use_pdl)
    _ok(_tree_calls()[2](args, _raw_stream(dev)), "tenzo_cuda_kv8_accept")
    return accepted, following, path


def kv8_take_errors() -> int:
    """Error flags of the kernels on trees and bounded caches since the last call (1: a wait was given up, 2: an index out of range), -1 if the query failed; waits for
    all streams of the device."""
    return int(load_library().tenzo_cuda_kv8_take_errors())
