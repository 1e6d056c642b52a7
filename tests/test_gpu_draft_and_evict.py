"""Speculative decoding over INT8 caches of a bounded number of tokens, step after step: the drafted nodes are stored, attended to, weighed and accepted, and the caches cut
back, so that places and positions part. Every step against numpy: rows, positions, paths and lengths bit for bit, the attention's results and weights within their bounds."""
import numpy as np
import pytest
import torch
import kv8_reference as ref
from gpu_helpers import dev, host

pytestmark = pytest.mark.gpu

N_Q, N_KV, LAYERS, SLOTS, ROPE = 12, 3, 2, 16, 1024


class Run:
    """The device's state, and what a step draws: rows, tokens and trees."""

    def __init__(self, lengths, nodes, keep, recent, steps):
        rng = np.random.default_rng(nodes * 1000 + keep)
        self.keep, self.recent, self.nodes = keep, recent, nodes
        self.columns = (max(max(lengths), keep) + nodes + SLOTS - 1) // SLOTS
        self.c = c = ref.Caches(rng, len(lengths), self.columns, LAYERS, N_KV, SLOTS)
        for s, n in enumerate(lengths):
            c.fill(rng, s, range(n))
            b, o = c.at(s, np.arange(n))
            c.weight[b, :, :, o], c.position[b, :, :, o] = rng.random((n, LAYERS, N_KV)), np.arange(n)[:, None, None]
        self.lengths, self.cos_sin, self.S = list(lengths), ref.rope(ROPE), len(lengths)
        self.steps = []
        rows = self.S * nodes
        for step in range(steps):
            parents = [[-1] + [int(rng.integers(max(0, i - 3), i)) for i in range(1, nodes)] for _ in range(self.S)]
            self.steps.append(dict(parents=np.array(parents, np.int32), count=np.array([max(1, nodes - 2 * ((s + step) % 3)) if s != step else 0 for s in range(self.S)], np.int32),
                                   token=rng.integers(0, 3, (self.S, nodes)).astype(np.int32), chosen=rng.integers(0, 3, (self.S, nodes)).astype(np.int32),
                                   q=[rng.standard_normal((rows, N_Q * 128)).astype(np.float32) for _ in range(LAYERS)],
                                   k=[rng.standard_normal((rows, N_KV * 128)).astype(np.float32) for _ in range(LAYERS)],
                                   v=[rng.standard_normal((rows, N_KV * 128)).astype(np.float32) for _ in range(LAYERS)]))
            for d in self.steps[-1:]:
                d["depth"] = np.zeros((self.S, nodes), np.int32)
                d["sees"] = []
                for s in range(self.S):
                    for i in range(1, nodes):
                        d["depth"][s, i] = d["depth"][s, parents[s][i]] + 1
                    d["sees"] += ref.ancestors(parents[s])
                d["mask"] = ref.masks(d["sees"], nodes, (nodes + 31) // 32)

    def device(self):
        from tenzo_b200 import kernels
        state = {n: dev(getattr(self.c, n)) for n in self.c.POOLS} | dict(length=dev(np.array(self.lengths, np.int32)), position_next=dev(np.array(self.lengths, np.int32)))
        cache = kernels.Kv8Cache(*(state[n] for n in ("k", "v", "sk", "sv")), dev(self.c.table))
        return state, cache, [{n: [dev(x) for x in y] if isinstance(y, list) else dev(y) for n, y in d.items() if n != "sees"} for d in self.steps], [dev(x) for x in self.cos_sin]

    def step(self, state, cache, d, rope):
        """A model's step: all on the device, no number read back."""
        from tenzo_b200 import kernels
        node = torch.arange(self.nodes, dtype=torch.int32, device="cuda")
        there = node < d["count"][:, None]
        place = torch.where(there, state["length"][:, None] + node, -1).to(torch.int32).flatten()
        rope_pos = (state["position_next"][:, None] + d["depth"]).to(torch.int32).flatten()
        seq = torch.arange(self.S, dtype=torch.int32, device="cuda").repeat_interleave(self.nodes)
        turn = dict(rope_pos=rope_pos, rope_cos=rope[0], rope_sin=rope[1])
        got = dict(out=[], lse=[])
        for layer in range(LAYERS):
            kernels.kv8_append(d["k"][layer], d["v"][layer], cache, place, layer=layer, seq=seq, weight=state["weight"], position=state["position"], **turn)
            a = dict(layer=layer, n_q=N_Q, nodes=self.nodes, count=d["count"], mask=d["mask"], **turn)
            out, lse = kernels.attention_tree(d["q"][layer], cache, state["length"], want_lse=True, **a)
            kernels.kv8_weigh(d["q"][layer], lse, cache, state["weight"], state["length"], **a)
            got["out"].append(out)
            got["lse"].append(lse)
        got["weighed"] = state["weight"].clone()
        got["accepted"], got["next"], got["path"] = kernels.kv8_accept(cache, d["token"], d["parents"], d["chosen"], state["length"], count=d["count"], weight=state["weight"],
                                                                       position=state["position"])
        state["position_next"] += got["accepted"]
        grown = state["length"] + got["accepted"]
        state["length"].copy_(kernels.kv8_evict(cache, state["weight"], state["position"], grown, keep=self.keep, protect_from=state["position_next"] - self.recent))
        return got

    def check_step(self, d, position, got):
        """The same in numpy; the weights then go on from the device's, whose order the eviction follows."""
        c, cos, sin = self.c, *self.cos_sin
        slack = np.zeros(c.weight.shape)
        want = c.weight.astype(np.float64)
        for layer in range(LAYERS):
            out, lse = (host(got[n][layer]).astype(np.float64) for n in ("out", "lse"))
            for s in range(self.S):
                n, rows = int(d["count"][s]), slice(s * self.nodes, s * self.nodes + int(d["count"][s]))
                at = position[s] + d["depth"][s, :n]
                b, o = c.at(s, self.lengths[s] + np.arange(n))
                for i in range(n):
                    r = s * self.nodes + i
                    c.k[b[i], layer, :, o[i]], c.sk[b[i], layer, :, o[i]] = ref.quantise(ref.rotate32(d["k"][layer][r].reshape(N_KV, 128), cos[at[i]], sin[at[i]]))
                    c.v[b[i], layer, :, o[i]], c.sv[b[i], layer, :, o[i]] = ref.quantise(d["v"][layer][r].reshape(N_KV, 128))
                c.weight[b, layer, :, o], c.position[b, layer, :, o], want[b, layer, :, o] = 0, at[:, None], 0
                end = slice(rows.stop, (s + 1) * self.nodes)
                assert (out[end] == 0).all() and np.isneginf(lse[end]).all()
                if n == 0:
                    continue
                w_out, w_lse, bound, lse_bound, weights = ref.tree(d["q"][layer][rows], c, layer, N_Q, (s, self.lengths[s]), d["sees"][rows], [(cos[p], sin[p]) for p in at])
                assert (np.abs(out[rows] - w_out) <= bound).all() and (np.abs(lse[rows] - w_lse) <= lse_bound).all()
                b, o = c.at(s, np.arange(weights.shape[1]))
                for h in range(N_KV):
                    want[b, layer, h, o] += weights[h]
                    # as in the weights' own test: what the exponentials' arguments are off by, and sums in fp32
                    slack[b, layer, h, o] += weights[h] * (2 * lse_bound.max() + (16 + n * N_Q / N_KV / 8) * 2.0 ** -24)
        weighed = host(got["weighed"])
        assert (np.abs(weighed - want) <= slack + 2.0 ** -23 * np.abs(want)).all()
        c.weight[...] = weighed
        new = []
        for s in range(self.S):
            n = int(d["count"][s])
            path, following = ref.accept(c, s, self.lengths[s], d["token"][s, :n], d["parents"][s, :n], d["chosen"][s, :n])
            assert host(got["path"])[s].tolist() == path + [-1] * (self.nodes - len(path)) and int(got["next"][s]) == following and int(got["accepted"][s]) == len(path)
            position[s] += len(path)
            new.append(ref.evict(c, s, self.lengths[s] + len(path), self.keep, position[s] - self.recent))
        self.lengths = new


@pytest.mark.parametrize("lengths,nodes,keep,recent", [([150, 20, 149, 0], 12, 150, 8), ([70, 71, 72], 40, 72, 30), ([5, 0], 1, 6, 1)])
def test_steps(cuda_lib, lengths, nodes, keep, recent):
    from tenzo_b200 import kernels
    run = Run(lengths, nodes, keep, recent, steps=5)
    state, cache, steps, rope = run.device()
    position = list(lengths)
    for i, d in enumerate(steps):
        got = run.step(state, cache, d, rope)
        run.check_step(run.steps[i], position, got)
        assert host(state["length"]).tolist() == run.lengths and host(state["position_next"]).tolist() == position
        assert run.c.same(type("", (), {n: host(state[n]) for n in run.c.POOLS})()) == []
    assert kernels.kv8_take_errors() == 0


def test_steps_in_a_graph(cuda_lib):
    """One capture, replayed with the next step's rows in the same buffers, gives the bits of the steps one by one."""
    run = Run([90, 31, 140], 16, 120, 20, steps=4)
    state, cache, steps, rope = run.device()
    again, cache2, _, _ = run.device()
    buffers = {n: [torch.empty_like(x) for x in y] if isinstance(y, list) else torch.empty_like(y) for n, y in steps[0].items()}

    def put(d):
        for n, y in d.items():
            for to, x in zip(buffers[n], y) if isinstance(y, list) else [(buffers[n], y)]:
                to.copy_(x)

    run.step(state, cache, steps[0], rope)
    put(steps[0])
    run.step(again, cache2, buffers, rope)                                    # (also the first use of each kernel)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run.step(again, cache2, buffers, rope)
    for d in steps[1:]:
        run.step(state, cache, d, rope)
        put(d)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(state[n].view(torch.uint8), again[n].view(torch.uint8)) for n in state)
