"""Forking the 4-bit cache to the beams that go on, and a whole beam search: append, attention, selection, reordering, step after step."""
import numpy as np
import pytest
import torch
import kv4_reference as ref
from gpu_helpers import Guarded, dev, host

pytestmark = pytest.mark.gpu


def beams_setup(rng, groups, beams, columns, layers, n_kv):
    blocks = groups * beams * columns + 1
    table = rng.permutation(blocks)[: groups * beams * columns].astype(np.int32).reshape(groups * beams, columns)
    return table, rng.integers(0, 256, (blocks, layers, n_kv, 2, 16, 80), dtype=np.uint8)


@pytest.mark.parametrize("groups,beams,lengths,layers,n_kv", [
    (1, 1, [5], 1, 1), (1, 4, [0], 2, 3), (2, 4, [16, 17], 3, 5), (3, 32, [31, 1, 47], 1, 2), (5, 7, [15, 32, 33, 48, 20], 2, 1), (1, 2, [40], 30, 5), (40, 3, [25] * 40, 4, 8),
])
def test_reorder(cuda_lib, groups, beams, lengths, layers, n_kv):
    from tenzo_b200 import kernels
    rng = np.random.default_rng(groups * 100 + beams)
    table, pool = beams_setup(rng, groups, beams, 3, layers, n_kv)
    table[:, 0] = table[0, 0] if groups == 1 and lengths[0] >= 16 else table[:, 0]              # a shared full block
    length = np.array(lengths, np.int32)
    for kind in ("random", "one", "same", "turned", "last"):
        parent = {"random": rng.integers(0, beams, (groups, beams)), "one": np.zeros((groups, beams)), "same": np.tile(np.arange(beams), (groups, 1)),
                  "turned": np.tile(np.arange(beams)[::-1], (groups, 1)), "last": np.full((groups, beams), beams - 1)}[kind].astype(np.int32)
        g = Guarded()
        d_pool, d_out = g.empty(pool.shape, torch.uint8, dev(pool)), g.empty(table.shape, torch.int32)
        kernels.kv4_reorder(d_pool, dev(table), dev(parent), dev(length), out=d_out)
        want_table, want_pool = ref.reorder(pool, table, parent, length)
        assert np.array_equal(host(d_out), want_table), kind
        assert np.array_equal(host(d_pool), want_pool), kind
        g.check()
    assert kernels.kv4_take_errors() == 0


def test_reorder_refuses_on_the_device(cuda_lib):
    """A parent, a length or a block out of range: that group (or copy) is left out, the others go on, the flag is up."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(1)
    groups, beams = 6, 4
    table, pool = beams_setup(rng, groups, beams, 3, 2, 2)
    parent = np.tile(np.array([1, 1, 2, 1], np.int32), (groups, 1))
    length = np.array([20, 20, -1, 49, 48, 20], np.int32)
    parent[1, 2] = 4
    parent[5, 0] = -1
    d_pool = dev(pool)
    out = kernels.kv4_reorder(d_pool, dev(table), dev(parent), dev(length))
    assert kernels.kv4_take_errors() == 2
    own = np.tile(np.arange(beams, dtype=np.int32), (groups, 1))
    fine = np.array([True, False, False, False, True, False])
    want_table, want_pool = ref.reorder(pool, table, np.where(fine[:, None], parent, own), np.where(length < 0, 0, length % 49).astype(np.int32))
    assert np.array_equal(host(out), want_table) and np.array_equal(host(d_pool), want_pool)
    broken = table.copy()
    broken[1, 1] = len(pool)                                            # the source of group 0's copies
    d_pool = dev(pool)
    out = kernels.kv4_reorder(d_pool, dev(broken), dev(np.tile(parent[:1], (groups, 1))), dev(np.full(groups, 20, np.int32)))
    assert kernels.kv4_take_errors() == 2
    want_table, _ = ref.reorder(pool, table, np.tile(parent[:1], (groups, 1)), np.full(groups, 20))
    want_table[want_table == table[1, 1]] = len(pool)
    _, want_pool = ref.reorder(pool, table, np.concatenate([own[:1], np.tile(parent[:1], (groups - 1, 1))]), np.full(groups, 20))
    assert np.array_equal(host(out), want_table) and np.array_equal(host(d_pool), want_pool)


def test_selection_and_reordering_overlapped(cuda_lib):
    """Selection, then the reordering that reads its parents, launched to overlap, many times over: nothing is read before the kernel in front has written it."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(2)
    groups, beams, vocab = 2, 4, 211
    table, pool = beams_setup(rng, groups, beams, 3, 1, 2)
    d_table, d_pool, length = dev(table), dev(pool), torch.full((groups,), 21, dtype=torch.int32, device="cuda")
    logits = [rng.standard_normal((groups * beams, vocab)).astype(np.float32) for _ in range(16)]
    scores = np.zeros(groups * beams, np.float32)
    want = []
    for x in logits:
        parent, token, _ = ref.select(x, scores, beams, beams)
        want.append((parent, token, *ref.reorder(pool, table, parent.astype(np.int32), np.full(groups, 21))))
    d_logits, d_scores = [dev(x) for x in logits], dev(scores)
    got = []
    for i in range(400):
        p = d_pool.clone()
        parent, token, _ = kernels.beam_select(d_logits[i % 16], d_scores, beams=beams, k=beams, use_pdl=True)
        got.append((parent, token, kernels.kv4_reorder(p, d_table, parent, length, use_pdl=True), p))
    for i, g in enumerate(got):
        assert all(np.array_equal(host(a), b) for a, b in zip(g, want[i % 16])), i


@pytest.mark.parametrize("pdl", [False, True])
def test_beam_search(cuda_lib, pdl):
    """Two requests with four beams, prompts that end inside a block and at its end, 40 steps: the beams' tokens are those of a search that
    keeps every beam's keys and values apart. The model is one layer: embedding rows as q|k|v, attention, a product with the vocabulary."""
    from tenzo_b200 import kernels
    rng = np.random.default_rng(11)
    groups, beams, n_q, n_kv, vocab, steps, eos = 2, 4, 4, 2, 211, 40, 7
    prompts = [rng.integers(0, vocab, n) for n in (21, 32)]
    width = (n_q + 2 * n_kv) * 128
    embed = rng.standard_normal((vocab, width)).astype(np.float32)
    head = (rng.standard_normal((n_q * 128, vocab)) * 0.35).astype(np.float32)
    length = np.array([len(p) for p in prompts], np.int32)
    most = int(length.max()) + steps + 1
    columns = (most + 15) // 16
    cos, sin = ref.rope(columns * 16)
    rows = groups * beams
    blocks = rows * columns
    table = rng.permutation(blocks).astype(np.int32).reshape(rows, columns)
    pool = torch.zeros(blocks, 1, n_kv, 2, 16, 80, dtype=torch.uint8, device="cuda")
    d_embed, d_head, d_cos, d_sin, d_table = dev(embed), dev(head), dev(cos), dev(sin), dev(table)

    # ---- the search that keeps everything apart
    def kv_rows(tokens, start):
        x = embed[tokens]
        at = np.arange(start, start + len(tokens))
        k = ref.rotate(x[:, n_q * 128: (n_q + n_kv) * 128].reshape(-1, n_kv, 128), cos[at][:, None], sin[at][:, None])
        v = x[:, (n_q + n_kv) * 128:].reshape(-1, n_kv, 128)
        return [ref.values(ref.quantise(y)).transpose(1, 0, 2) for y in (k, v)]

    class Beam:
        def __init__(self, k, v, tokens):
            self.k, self.v, self.tokens = k, v, tokens

    state = []
    for p in prompts:
        k, v = kv_rows(p, 0)
        state.append([Beam(k, v, list(p)) for _ in range(beams)])

    # ---- the prompts into the first beam's blocks, then forked
    for g, p in enumerate(prompts):
        x = d_embed[torch.from_numpy(p).cuda()]
        n = len(p)
        kernels.kv4_append(x[:, n_q * 128: (n_q + n_kv) * 128], x[:, (n_q + n_kv) * 128:], pool, torch.arange(n, dtype=torch.int32, device="cuda"), layer=0,
                           block_table=d_table, seq=torch.full((n,), g * beams, dtype=torch.int32, device="cuda"), rope_cos=d_cos, rope_sin=d_sin)
    d_length = dev(length)
    other = torch.empty_like(d_table)
    kernels.kv4_reorder(pool, d_table, torch.zeros(groups, beams, dtype=torch.int32, device="cuda"), d_length, out=other)
    d_table, other = other, d_table
    scores = torch.tensor([0.0] + [-torch.inf] * (beams - 1), device="cuda").repeat(groups)
    want_scores = host(scores).astype(np.float32)
    finished = torch.zeros(rows, dtype=torch.int32, device="cuda")
    tokens = torch.from_numpy(np.repeat([p[-1] for p in prompts], beams).astype(np.int64)).cuda()

    for step in range(steps):
        # the token at the end of each beam is the query; from the second step on it is appended first
        x = d_embed[tokens]
        if step:
            pos = d_length.repeat_interleave(beams)
            kernels.kv4_append(x[:, n_q * 128: (n_q + n_kv) * 128], x[:, (n_q + n_kv) * 128:], pool, pos, layer=0, block_table=d_table, rope_cos=d_cos, rope_sin=d_sin,
                               use_pdl=pdl)
            d_length = d_length + 1
        pos = d_length.repeat_interleave(beams) - 1
        out = kernels.attention_kv4(x[:, : n_q * 128], pool, pos, layer=0, n_q=n_q, block_table=d_table, rope_cos=d_cos, rope_sin=d_sin, max_len=most, use_pdl=False)
        logits = (out.double() @ d_head.double()).float()
        parent, token, score = kernels.beam_select(logits, scores, beams=beams, k=beams, finished=finished, eos=eos, use_pdl=pdl)
        kernels.kv4_reorder(pool, d_table, parent, d_length, out=other, use_pdl=pdl)
        d_table, other = other, d_table
        flat = (parent.long() + beams * torch.arange(groups, device="cuda")[:, None]).flatten()
        finished = (finished[flat].bool() | (token.flatten() == eos)).to(torch.int32)
        scores, tokens = score.flatten(), token.flatten().long()

        want_logits = np.empty((rows, vocab))
        for g in range(groups):
            for b, beam in enumerate(state[g]):
                last = beam.tokens[-1]
                if step:
                    k, v = kv_rows(np.array([last]), len(beam.tokens) - 1)
                    beam.k, beam.v = np.concatenate([beam.k, k], 1), np.concatenate([beam.v, v], 1)
                n = beam.k.shape[1]
                o, _ = ref.attention(embed[last][: n_q * 128].reshape(n_q, 128), beam.k, beam.v, cos[n - 1], sin[n - 1])
                want_logits[g * beams + b] = o.reshape(-1) @ head.astype(np.float64)
        done = np.array([eos in beam.tokens[len(prompts[g]):] for g in range(groups) for beam in state[g]]).astype(np.int32)
        wp, wt, ws = ref.select(want_logits.astype(np.float32), want_scores, beams, beams, done, eos)
        assert np.array_equal(host(parent), wp) and np.array_equal(host(token), wt), step
        live = np.isfinite(ws)
        assert np.allclose(host(score)[live], ws[live], rtol=1e-5, atol=1e-5)
        state = [[Beam(state[g][p].k, state[g][p].v, state[g][p].tokens + [int(t)]) for p, t in zip(wp[g], wt[g])] for g in range(groups)]
        want_scores = host(score).reshape(-1)                            # the sums go on from the same numbers
    assert kernels.kv4_take_errors() == 0
    last = host(d_length)
    for g in range(groups):                                              # and the caches hold the beams' own rows
        for b, beam in enumerate(state[g]):
            n = int(last[g])
            k, v = kernels.kv4_read(pool, torch.arange(n, dtype=torch.int32, device="cuda"), layer=0, block_table=d_table,
                                    seq=torch.full((n,), g * beams + b, dtype=torch.int32, device="cuda"))
            assert np.array_equal(host(k).reshape(n, n_kv, 128), beam.k.transpose(1, 0, 2).astype(np.float32))
            assert np.array_equal(host(v).reshape(n, n_kv, 128), beam.v.transpose(1, 0, 2).astype(np.float32))
