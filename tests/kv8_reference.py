"""What the calls on trees and bounded caches over the INT8 caches do, in numpy and 64 bits."""
import numpy as np


def rope(length, theta=10000.0):
    at = np.arange(length)[:, None] * theta ** (-np.arange(64) / 64)
    return np.cos(at).astype(np.float32), np.sin(at).astype(np.float32)


def rotate(x, c, s):
    """x [..., 128], pairs (i, i + 64): in 64 bits."""
    a, b = x[..., :64].astype(np.float64), x[..., 64:].astype(np.float64)
    c, s = np.float64(c), np.float64(s)
    return np.concatenate([a * c - b * s, a * s + b * c], -1)


def rotate32(x, c, s):
    """The same as the kernels round it: one product to fp32, the other fused with the sum."""
    a, b = x[..., :64], x[..., 64:]
    wide = np.float64
    return np.concatenate([(a.astype(wide) * wide(c) - (b * s).astype(wide)).astype(np.float32), (a.astype(wide) * wide(s) + (b * c).astype(wide)).astype(np.float32)], -1)


def quantise(x):
    """(codes, scale) of rows [..., 128], every step rounded to fp32; halves away from zero."""
    f = np.float32
    scale = np.maximum(np.abs(x).max(-1), f(1e-8)) * (f(1) / f(127))
    code = (x * (f(1) / scale)[..., None]).astype(np.float64)
    return np.clip(np.copysign(np.floor(np.abs(code) + 0.5), code), -128, 127).astype(np.int8), scale


class Caches:
    """Pools of anything, NaN among the scales of places that nobody owns, and a table; `slots` per block."""

    def __init__(self, rng, sequences, columns, layers, n_kv, slots, spare=2):
        self.n_blocks, self.layers, self.n_kv, self.slots = sequences * columns + spare, layers, n_kv, slots
        shape = (self.n_blocks, layers, n_kv, slots)
        self.k, self.v = (rng.integers(-128, 128, shape + (128,), dtype=np.int8) for _ in range(2))
        self.sk, self.sv = (np.full(shape, np.nan, np.float32) for _ in range(2))
        self.table = rng.permutation(self.n_blocks)[: sequences * columns].astype(np.int32).reshape(sequences, columns)
        self.weight = rng.random(shape).astype(np.float32)
        self.position = rng.integers(0, 1 << 20, shape).astype(np.int32)

    POOLS = ("k", "v", "sk", "sv", "weight", "position")

    def copy(self):
        c = object.__new__(Caches)
        c.__dict__.update({n: x.copy() if isinstance(x, np.ndarray) else x for n, x in self.__dict__.items()})
        return c

    def at(self, seq, place):
        return self.table[seq, place // self.slots], place % self.slots

    def fill(self, rng, seq, places, low=0.01, high=0.03):
        """Values of a quantiser: codes of a normal distribution, scales between `low` and `high`."""
        for t in places:
            b, o = self.at(seq, t)
            for code, scale in ((self.k, self.sk), (self.v, self.sv)):
                code[b, :, :, o] = np.clip(np.rint(rng.standard_normal((self.layers, self.n_kv, 128)) * 44), -127, 127)
                scale[b, :, :, o] = low + (high - low) * rng.random((self.layers, self.n_kv))

    def rows(self, which, layer, seq, kvh, n):
        """[n, 128] in 64 bits."""
        codes, scales = (self.k, self.sk) if which == "k" else (self.v, self.sv)
        b, o = self.at(seq, np.arange(n))
        return codes[b, layer, kvh, o].astype(np.float64) * scales[b, layer, kvh, o].astype(np.float64)[:, None]

    def same(self, other):
        return [n for n in self.POOLS if getattr(self, n).tobytes() != getattr(other, n).tobytes()]


def ancestors(parents):
    seen = []
    for i, p in enumerate(parents):
        seen.append((seen[p] if p >= 0 else set()) | {i})
    return seen


def masks(sees, nodes, words):
    """int32 [len(sees), words] from sets of nodes."""
    out = np.zeros((len(sees), words), np.uint32)
    for i, s in enumerate(sees):
        for j in s:
            out[i, j // 32] |= np.uint32(1 << (j % 32))
    return out.view(np.int32)


def tree(q, caches, layer, n_q, start, sees, turn=None):
    """One sequence (start, table row in `caches`): q [nodes, n_q*128]; sees: for each node the set of nodes; turn: (cos, sin) rows per node. start is (table row, tokens).
    Returns out, lse and the bound of |out - these| that the kernel's roundings allow."""
    seq, cached = start
    nodes, group = len(sees), n_q // caches.n_kv
    n = cached + nodes
    out, lse = np.zeros((len(q), n_q, 128)), np.full((len(q), n_q), -np.inf)
    bound, lse_bound = np.zeros((len(q), n_q)), np.zeros((len(q), n_q))
    weight = np.zeros((caches.n_kv, n))
    for h in range(caches.n_kv):
        key, value = caches.rows("k", layer, seq, h, n), caches.rows("v", layer, seq, h, n)
        for i in range(nodes):
            x = q[i].reshape(n_q, 128)[h * group: (h + 1) * group]
            x = rotate(x, *turn[i]) if turn is not None else x.astype(np.float64)
            places = np.array(list(range(cached)) + sorted(cached + j for j in sees[i] if j < nodes), dtype=int)
            if not len(places):
                continue
            for g in range(group):
                s = key[places] @ x[g] / np.sqrt(128)
                top = s.max()
                e = np.exp(s - top)
                head = h * group + g
                out[i, head] = e @ value[places] / e.sum()
                lse[i, head] = top + np.log(e.sum())
                weight[h, places] += e / e.sum()
                # the query: half a step of 2^-21 of its largest; each product, sum and the exponential's argument: some steps of fp32 of the sum of magnitudes;
                # a weight: half a step of 2^-26 of the largest, counted with scales that may be half the largest
                reach = (np.abs(key[places]) @ np.abs(x[g])).max() / np.sqrt(128)
                ds = 2.0 ** -22 * np.abs(x[g]).max() * np.abs(key[places]).sum(-1).max() / np.sqrt(128) + 24 * 2.0 ** -24 * (reach + 1)
                sums = (16 + len(places) / 16) * 2.0 ** -24
                most = np.abs(value[places]).max()
                bound[i, head] = most * (2 * ds + sums + len(places) * 2.0 ** -26)
                lse_bound[i, head] = ds + sums + 4 * 2.0 ** -24 * (1 + abs(lse[i, head]))
    return out.reshape(len(q), -1), lse, np.repeat(bound, 128, 1), lse_bound, weight


def evict(c, seq, n, keep, protect_from):
    """In place; the sequence's new length."""
    if n <= keep:
        return n
    b, o = c.at(seq, np.arange(n))
    for layer in range(c.layers):
        for h in range(c.n_kv):
            w = c.weight[b, layer, h, o].copy()
            w[np.isnan(w)] = -np.inf
            if protect_from is not None:
                w[c.position[b, layer, h, o] >= protect_from] = np.inf
            stays = np.zeros(n, bool)
            stays[np.argsort(-w, kind="stable")[:keep]] = True
            far, holes = np.flatnonzero(stays[keep:]) + keep, np.flatnonzero(~stays[:keep])
            for name in c.POOLS:
                x = getattr(c, name)
                x[b[holes], layer, h, o[holes]] = x[b[far], layer, h, o[far]].copy()
    return keep


def accept(c, seq, start, token, parent, chosen):
    """In place; (path, next token)."""
    path = [0] if len(token) else []
    while path:
        cur = path[-1]
        on = [j for j in range(cur + 1, len(token)) if parent[j] == cur and token[j] == chosen[cur]]
        if not on:
            break
        path.append(on[0])
    if path:
        (fb, fo), (tb, to) = c.at(seq, start + np.array(path)), c.at(seq, start + np.arange(len(path)))
        for name in c.POOLS:
            x = getattr(c, name)
            x[tb, :, :, to] = x[fb, :, :, fo].copy()
    return path, (chosen[path[-1]] if path else -1)
