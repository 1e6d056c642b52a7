"""Received weight of drafted steps that does not count refused nodes: weighed behind the acceptance, for the accepted path as a chain. Against 64 bits over the accepted nodes alone, and against the same
tokens decoded without any draft."""
import numpy as np
import pytest
import torch
import kv8_reference as ref
from gpu_helpers import dev, host

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths,nodes,n_q,n_kv", [([150, 0, 700, 33], 12, 12, 3), ([90, 1000], 40, 8, 2), ([5], 1, 4, 1), ([260, 128], 70, 16, 2)])
def test_refused_nodes_do_not_count(cuda_lib, lengths, nodes, n_q, n_kv):
    from tenzo_b200 import kernels
    rng = np.random.default_rng(nodes)
    S = len(lengths)
    c = ref.Caches(rng, S, (max(lengths) + nodes + 15) // 16, 1, n_kv, 16)
    for s, n in enumerate(lengths):
        c.fill(rng, s, range(n))
    parent = np.array([[-1] + [int(rng.integers(max(0, i - 3), i)) for i in range(1, nodes)] for _ in range(S)], np.int32)
    token, chosen = (rng.integers(0, 2, (S, nodes)).astype(np.int32) for _ in range(2))
    count = np.array([nodes - 3 * (s % 2) * (nodes > 6) for s in range(S)], np.int32)
    depth = np.zeros((S, nodes), np.int32)
    for i in range(1, nodes):
        depth[:, i] = depth[np.arange(S), parent[:, i]] + 1
    sees = [x for s in range(S) for x in ref.ancestors(parent[s])]
    q, k, v = (rng.standard_normal((S * nodes, h * 128)).astype(np.float32) for h in (n_q, n_kv, n_kv))
    cos, sin = ref.rope(max(lengths) + nodes)
    place = np.where(np.arange(nodes) < count[:, None], np.array(lengths)[:, None] + np.arange(nodes), -1).astype(np.int32).flatten()
    pos = (np.array(lengths)[:, None] + depth).astype(np.int32).flatten()
    start, qd, kd, vd = dev(np.array(lengths, np.int32)), dev(q), dev(k), dev(v)
    seq = torch.arange(S, dtype=torch.int32, device="cuda").repeat_interleave(nodes)
    turn = dict(rope_cos=dev(cos), rope_sin=dev(sin))

    def pools():
        return {n: dev(getattr(c, n)) for n in c.POOLS}

    state = pools()
    cache = kernels.Kv8Cache(*(state[n] for n in ("k", "v", "sk", "sv")), dev(c.table))
    kernels.kv8_append(kd, vd, cache, dev(place), layer=0, seq=seq, rope_pos=dev(pos), weight=state["weight"], position=state["position"], **turn)
    out, lse = kernels.attention_tree(qd, cache, start, layer=0, n_q=n_q, nodes=nodes, count=dev(count), mask=dev(ref.masks(sees, nodes, (nodes + 31) // 32)), rope_pos=dev(pos), want_lse=True, **turn)
    accepted, _, path = kernels.kv8_accept(cache, dev(token), dev(parent), dev(chosen), start, count=dev(count), weight=state["weight"], position=state["position"])
    row = (path.clamp(min=0).long() + nodes * torch.arange(S, device="cuda")[:, None]).flatten()
    kernels.kv8_weigh(qd[row], lse[row], cache, state["weight"], start, layer=0, n_q=n_q, nodes=nodes, count=accepted, rope_pos=dev(pos)[row], **turn)

    # the accepted tokens alone, one step each, without a tree
    plain = pools()
    other = kernels.Kv8Cache(*(plain[n] for n in ("k", "v", "sk", "sv")), dev(c.table))
    line = host(path)
    for d in range(int(accepted.max())):
        node = torch.from_numpy(np.maximum(line[:, d], 0).astype(np.int64)).cuda() + nodes * torch.arange(S, device="cuda")
        there = dev((line[:, d] >= 0).astype(np.int32))
        at = torch.where(there > 0, start + d, -1).to(torch.int32)
        kernels.kv8_append(kd[node], vd[node], other, at, layer=0, weight=plain["weight"], position=plain["position"], **turn)
        _, one = kernels.attention_tree(qd[node], other, start + d, layer=0, n_q=n_q, nodes=1, count=there, want_lse=True, **turn)
        kernels.kv8_weigh(qd[node], one, other, plain["weight"], start + d, layer=0, n_q=n_q, nodes=1, count=there, **turn)
    got, want, exact = (host(state["weight"]).astype(np.float64), host(plain["weight"]).astype(np.float64), c.weight.astype(np.float64))
    moved = ref.Caches.copy(c)                                                  # codes as the device has them now
    for n in ("k", "v", "sk", "sv"):
        setattr(moved, n, host(state[n]))
    for s in range(S):
        m = int(accepted[s])
        nodes_of = line[s, :m]
        assert m >= 1 and (pos.reshape(S, nodes)[s, nodes_of] == lengths[s] + np.arange(m)).all()
        rows = s * nodes + nodes_of
        _, _, _, lse_bound, weights = ref.tree(q[rows], moved, 0, n_q, (s, lengths[s]), [set(range(i + 1)) for i in range(m)], [(cos[p], sin[p]) for p in pos[rows]])
        b, o = c.at(s, np.arange(lengths[s] + m))
        exact[b[lengths[s]:], :, :, o[lengths[s]:]] = 0
        for h in range(n_kv):
            exact[b, 0, h, o] += weights[h]
            # as in the weights' own test: what arguments are off by in the attention and again here, sums and the old weight in fp32
            slack = weights[h] * (2 * lse_bound.max() + (16 + m * n_q / n_kv / 8) * 2.0 ** -24) + 2.0 ** -23 * exact[b, 0, h, o]
            assert (np.abs(got[b, 0, h, o] - exact[b, 0, h, o]) <= slack).all()
            # one step each: an addition to memory a token instead of one in all
            assert (np.abs(want[b, 0, h, o] - exact[b, 0, h, o]) <= slack + m * 2.0 ** -24 * exact[b, 0, h, o]).all()
    assert kernels.kv8_take_errors() == 0
