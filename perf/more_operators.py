"""Operators of drafted trees of tokens, and of caches of a bounded number of tokens, over the INT8 key-value caches: storing rows whose rotary
position is not their place, attention of a tree's nodes, the tokens of a tree that the model agrees with, the attention weight that each
cached token has received, and the eviction of the tokens that received least.

A cache is int8 [block][layer][kv head][slots][128] for keys and for values, each with fp32 scales [block][layer][kv head][slots]; the token at
place t of a sequence lies in block block_table[sequence][t / slots], slot t % slots. Sixteen slots a block make the block pools, one block a
sequence the contiguous cache. What eviction goes by, a weight (fp32) and a position (int32) for each cached token and kv head, is laid out as the scales are.

`own` says which side run() takes: the operators in elementary torch operations, or the framework's kernels.
"""
import math

import numpy as np
import torch

own = False

HD = 128


def listed():
    return [
        # One layer's rows of a batch of drafted trees, and a ragged batch of prompts, some rows being padding.
        {"name": "append_tree_16x32", "kind": "append", "sequences": 16, "nodes": 32, "context": 1500, "n_kv": 5, "slots": 16, "padded": False},
        {"name": "append_ragged_8x1000", "kind": "append", "sequences": 8, "nodes": 1000, "context": 333, "n_kv": 8, "slots": 16, "padded": True},
        # One conversation with eight drafted tokens; a server's step without any; with sixteen each over ragged contexts; with large trees over long ones.
        {"name": "tree_1x8", "kind": "tree", "sequences": 1, "nodes": 8, "context": 1000, "ragged": False, "n_q": 20, "n_kv": 5, "slots": 16},
        {"name": "tree_64x1", "kind": "tree", "sequences": 64, "nodes": 1, "context": 8192, "ragged": False, "n_q": 20, "n_kv": 5, "slots": 16},
        {"name": "tree_64x16_ragged", "kind": "tree", "sequences": 64, "nodes": 16, "context": 4095, "ragged": True, "n_q": 20, "n_kv": 5, "slots": 16},
        {"name": "tree_16x64", "kind": "tree", "sequences": 16, "nodes": 64, "context": 8192, "ragged": False, "n_q": 20, "n_kv": 5, "slots": 16},
        # The weights of a decode step of many sequences, and of the last rows of a few prompts over contiguous caches.
        {"name": "weigh_64x1", "kind": "weigh", "sequences": 64, "nodes": 1, "context": 4096, "ragged": False, "n_q": 20, "n_kv": 5, "slots": 16},
        {"name": "weigh_7x33", "kind": "weigh", "sequences": 7, "nodes": 33, "context": 6001, "ragged": True, "n_q": 32, "n_kv": 8, "slots": 6048},
        # A conversation cut back to its budget in all 30 layers, and a server's batch in some.
        {"name": "evict_1x2176", "kind": "evict", "sequences": 1, "layers": 30, "n_kv": 5, "context": 2176, "keep": 2048, "recent": 256, "slots": 16},
        {"name": "evict_64x4224", "kind": "evict", "sequences": 64, "layers": 4, "n_kv": 5, "context": 4224, "keep": 4096, "recent": 512, "slots": 16},
        # The accepted tokens of one tree, and of a batch of trees, in all 30 layers.
        {"name": "accept_1x24", "kind": "accept", "sequences": 1, "nodes": 24, "layers": 30, "n_kv": 5, "context": 219, "slots": 16},
        {"name": "accept_64x32", "kind": "accept", "sequences": 64, "nodes": 32, "layers": 30, "n_kv": 5, "context": 1500, "slots": 16},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["append", "tree", "tree", "tree", "weigh", "evict", "accept"])
    n_q, n_kv = rng.choice([(20, 5), (20, 5), (32, 8), (16, 16), (40, 5), (12, 4), (7, 1), (32, 2), (6, 1)])
    contiguous = rng.random() < 0.25
    if kind == "append":
        sequences = _log_int(rng, 1, 64)
        nodes, context = _log_int(rng, 1, max(1, 8000 // sequences)), _log_int(rng, 1, 2000) - 1
        case = {"kind": kind, "sequences": sequences, "nodes": nodes, "context": context, "n_kv": min(n_kv, 8), "padded": rng.random() < 0.5}
        most = context + nodes
    elif kind in ("tree", "weigh"):
        sequences, nodes = _log_int(rng, 1, 64), rng.choice([1, 1, _log_int(rng, 2, 64), _log_int(rng, 2, 64), _log_int(rng, 65, 256)])
        cost = 16 * 8192 * 5 if kind == "tree" else 64 * 4096 * 5
        context = min(_log_int(rng, 1, 32768) - 1, cost // (sequences * n_kv), cost * 64 * 4 // (sequences * nodes * n_q))
        case = {"kind": kind, "sequences": sequences, "nodes": nodes, "context": context, "ragged": rng.random() < 0.6, "n_q": n_q, "n_kv": n_kv}
        most = context + nodes
    elif kind == "evict":
        layers, n_kv = rng.choice([(1, 5), (2, 1), (4, 5), (8, 8), (30, 5)])
        context = _log_int(rng, 16, 16384)
        keep = max(1, context - min(context - 1, _log_int(rng, 1, max(1, context // 2))))
        sequences = _log_int(rng, 1, max(1, min(64, 64 * 4 * 5 * 4224 // (layers * n_kv * context))))
        case = {"kind": kind, "sequences": sequences, "layers": layers, "n_kv": n_kv, "context": context, "keep": keep, "recent": _log_int(rng, 1, max(1, keep))}
        most = context
    else:
        layers, n_kv = rng.choice([(30, 5), (32, 8), (2, 1)])
        nodes, context = _log_int(rng, 2, 64), _log_int(rng, 1, 2000) - 1
        sequences = _log_int(rng, 1, min(64, max(1, 64 * 32 * 150 // (nodes * layers * n_kv))))
        case = {"kind": kind, "sequences": sequences, "nodes": nodes, "layers": layers, "n_kv": n_kv, "context": context}
        most = context + nodes
        contiguous = contiguous and sequences * layers * n_kv * most < 4000000
    case["slots"] = (most + 15) // 16 * 16 if contiguous else 16
    return case


# ---- sizes -------------------------------------------------------------------------------------------------------------
def _spread(most, count):
    """Lengths of a batch: from half of `most` to `most`, as in a server that admits requests one by one."""
    return [most - (i * 2654435761 >> 7) % max(1, most // 2 + 1) for i in range(count)]


def _lengths(case):
    """Tokens that the sequences hold when their caches are cut back: between the budget and the largest context, or still a little below."""
    gone = case["context"] - case["keep"]
    return [max(1, case["context"] - (i * 2654435761 >> 7) % (gone + gone // 4 + 1)) for i in range(case["sequences"])]


def _starts(case):
    return _spread(case["context"], case["sequences"]) if case.get("ragged", True) else [case["context"]] * case["sequences"]


def _counts(case):
    """Nodes that each tree really has."""
    n = case["nodes"]
    return [n - (s * 97) % (n // 3 + 1) if case.get("ragged", case["kind"] == "accept") else n for s in range(case["sequences"])]


def _parents(n, s):
    """A tree whose nodes go on from one of the last few in front of them: a main line with branches."""
    return [-1] + [max(0, i - 1 - (i * i * 7 + s * 3 + i) % 5) for i in range(1, n)]


def _path(n, s):
    """The nodes that the model agrees with: from the root towards the last node."""
    parents, line, i = _parents(n, s), [], n - 1
    while i >= 0:
        line.append(i)
        i = parents[i]
    line.reverse()
    return line[: max(1, len(line) - (s * 5) % len(line))]


def _append_rows(case):
    """(sequence, place, position) of each row; place -1 where the row is padding. The tokens of a tree are rotated by their depth, not their place."""
    rows = []
    for s in range(case["sequences"]):
        start = case["context"] - (s * 40503) % max(1, case["context"] // 2 + 1)
        real = case["nodes"] - (s * 97) % (case["nodes"] // 3 + 1) if case["padded"] else case["nodes"]
        rows += [(s, start + i if i < real else -1, start + i // 2) for i in range(case["nodes"])]
    return rows


def work(case):
    kind = case["kind"]
    if kind == "append":            # fp32 rows in, their bytes, scales, weight and position out
        rows = _append_rows(case)
        real = sum(p >= 0 for _, p, _ in rows)
        return {"bytes": real * case["n_kv"] * (2 * HD * 4 + 2 * (HD + 4) + 8) + 12 * len(rows), "flops": 10 * real * case["n_kv"] * 2 * HD}
    if kind in ("tree", "weigh"):
        starts, counts = _starts(case), _counts(case)
        cached = sum(a + n for a, n in zip(starts, counts))
        seen = sum(a * n + sum(_depths(n, s)) + n for s, (a, n) in enumerate(zip(starts, counts)))
        rows = sum(counts)
        q = rows * case["n_q"] * HD * 4
        if kind == "weigh":
            return {"bytes": cached * case["n_kv"] * (HD + 4 + 8) + q + 4 * rows * case["n_q"], "flops": 2 * seen * case["n_q"] * HD}
        return {"bytes": cached * case["n_kv"] * 2 * (HD + 4) + 2 * q, "flops": 4 * seen * case["n_q"] * HD}
    if kind == "evict":             # every token's weight and position, and the rows that change their places
        keep, recent, n = case["keep"], case["recent"], 0
        moved = 0
        for length in _lengths(case):
            gone = max(0, length - keep)
            late = min(recent, gone)
            n += length if gone else 0
            moved += late + int((gone - late) * max(0, keep - late) / max(1, length - late))
        return {"bytes": case["layers"] * case["n_kv"] * (8 * n + 2 * moved * (2 * (HD + 4) + 8)), "flops": 0}
    moved = 0
    for s, n in enumerate(_counts(case)):
        moved += sum(i != d for d, i in enumerate(_path(n, s)))
    return {"bytes": case["layers"] * case["n_kv"] * 2 * moved * (2 * (HD + 4) + 8) + 16 * case["sequences"] * case["nodes"], "flops": 0}


# ---- states ------------------------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _depths(n, s):
    depth = []
    for p in _parents(n, s):
        depth.append(0 if p < 0 else depth[p] + 1)
    return depth


def _masks(n, s, columns):
    """Bit j of row i: node i goes on from node j, or is it."""
    seen = []
    for i, p in enumerate(_parents(n, s)):
        seen.append((seen[p] if p >= 0 else 0) | 1 << i)
    return [[m >> 32 * w & 0xFFFFFFFF for w in range(columns)] for m in seen]


def _columns(tokens, slots):
    return (tokens + slots - 1) // slots


def _caches(g, blocks, layers, n_kv, slots):
    """Rows as quantising values near N(0, 1) leaves them, with scales of their own."""
    shape = (blocks, layers, n_kv, slots, HD)
    rows = [torch.randn(shape, generator=g, device="cuda", dtype=torch.float16).mul_(44).clamp_(-127, 127).to(torch.int8) for _ in range(2)]
    scales = [0.015 + 0.015 * torch.rand(shape[:-1], generator=g, device="cuda") for _ in range(2)]
    return rows + scales


def _table(g, sequences, columns):
    """Every sequence has blocks of its own, from anywhere in the pool."""
    return torch.randperm(sequences * columns, generator=g, device="cuda").to(torch.int32).view(sequences, columns)


def _rope(length):
    at = torch.arange(length, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-torch.arange(64, dtype=torch.float64, device="cuda") / 64)
    return at.cos().float(), at.sin().float()


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g, kind, slots = _generator(seed), case["kind"], case["slots"]
    s = {"case": case}
    if kind == "append":
        rows = _append_rows(case)
        s["seq"], s["place"], s["pos"] = (_ints([r[i] for r in rows]) for i in range(3))
        most = case["context"] + case["nodes"]
        columns = _columns(most, slots)
        s["table"] = _table(g, case["sequences"], columns)
        s["k"], s["v"], s["sk"], s["sv"] = _caches(g, case["sequences"] * columns, 1, case["n_kv"], slots)
        s["weight"] = torch.rand(s["sk"].shape, generator=g, device="cuda")
        s["position"] = torch.randint(0, most, s["sk"].shape, generator=g, device="cuda", dtype=torch.int32)
        s["cos"], s["sin"] = _rope(most)
        for name in ("new_k", "new_v"):     # values of a projection: some dims a good deal larger than the rest
            s[name] = torch.randn(len(rows), case["n_kv"] * HD, generator=g, device="cuda")
            s[name] *= torch.exp(0.7 * torch.randn(case["n_kv"] * HD, generator=g, device="cuda"))
        return s
    if kind in ("tree", "weigh"):
        starts, counts, nodes = _starts(case), _counts(case), case["nodes"]
        s["max_len"] = case["context"] + nodes
        columns, words = _columns(s["max_len"], slots), (nodes + 31) // 32
        s["table"] = _table(g, case["sequences"], columns)
        s["k"], s["v"], s["sk"], s["sv"] = _caches(g, case["sequences"] * columns, 1, case["n_kv"], slots)
        s["start"], s["count"] = _ints(starts), _ints(counts)
        masks, pos = [], []
        for i, a in enumerate(starts):
            masks += _masks(nodes, i, words)
            pos += [a + d for d in _depths(nodes, i)]
        s["mask"] = torch.from_numpy(np.array(masks, dtype=np.uint32).view(np.int32)).cuda()
        s["pos"] = _ints(pos)
        s["cos"], s["sin"] = _rope(s["max_len"])
        s["q"] = 1.5 * torch.randn(len(pos), case["n_q"] * HD, generator=g, device="cuda")
        if kind == "weigh":             # as the attention in front left it, and the weights of the steps before
            s["lse"] = _scores(s)[1]
            s["weight"] = 8 * torch.rand(s["sk"].shape, generator=g, device="cuda") ** 4
        return s
    sequences, layers, n_kv = case["sequences"], case["layers"], case["n_kv"]
    if kind == "evict":
        lengths = _lengths(case)
        columns = _columns(case["context"], slots)
        s["table"] = _table(g, sequences, columns)
        s["k"], s["v"], s["sk"], s["sv"] = _caches(g, sequences * columns, layers, n_kv, slots)
        s["length"], s["from"] = _ints(lengths), _ints([n + 1000 - case["recent"] for n in lengths])
        s["weight"] = 8 * torch.rand(s["sk"].shape, generator=g, device="cuda") ** 4
        # up to the budget in any order, as evictions leave them, and behind it the newest, in theirs; a thousand tokens were evicted before
        place = torch.arange(columns * slots, device="cuda")[None, None, None].expand(sequences, layers, n_kv, -1)
        key = torch.where(place < case["keep"], torch.rand(place.shape, generator=g, device="cuda") * case["keep"], place.float())
        position = torch.empty(place.shape, dtype=torch.int32, device="cuda").scatter_(-1, key.argsort(-1), (place + 1000).to(torch.int32))
        s["position"] = torch.empty(s["sk"].shape, dtype=torch.int32, device="cuda")
        s["position"][s["table"].long().flatten()] = position.unflatten(-1, (columns, slots)).permute(0, 3, 1, 2, 4).flatten(0, 1)
        return s
    starts, counts, nodes = _starts(case), _counts(case), case["nodes"]
    first = [a // slots for a in starts]
    columns = _columns(case["context"] + nodes, slots)
    own_blocks = [(i, c) for i, a in enumerate(starts) for c in range(first[i], _columns(a + nodes, slots))]
    blocks = torch.randperm(len(own_blocks), generator=g, device="cuda").to(torch.int32)     # those of the trees; the ones in front are not touched
    s["table"] = torch.zeros(sequences, columns, dtype=torch.int32, device="cuda")
    at = torch.tensor(own_blocks, device="cuda")
    s["table"][at[:, 0], at[:, 1]] = blocks
    s["k"], s["v"], s["sk"], s["sv"] = _caches(g, len(own_blocks), layers, n_kv, slots)
    s["weight"] = torch.rand(s["sk"].shape, generator=g, device="cuda")
    s["position"] = torch.randint(0, 4096, s["sk"].shape, generator=g, device="cuda", dtype=torch.int32)
    s["start"], s["count"] = _ints(starts), _ints(counts)
    s["parent"] = _ints([_parents(nodes, i) for i in range(sequences)])
    s["token"] = torch.randint(0, 128256, (sequences, nodes), generator=g, device="cuda", dtype=torch.int32)
    s["chosen"] = torch.randint(0, 128256, (sequences, nodes), generator=g, device="cuda", dtype=torch.int32)
    paths = [_path(n, i) for i, n in enumerate(counts)]
    links = torch.tensor([(i, a, b) for i, p in enumerate(paths) for a, b in zip(p, p[1:])] or [(0, 0, 0)], device="cuda")
    s["chosen"][links[:, 0], links[:, 1]] = s["token"][links[:, 0], links[:, 2]]
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------------
def run(state):
    kind, case = state["case"]["kind"], state["case"]
    if own:
        from tenzo_b200 import kernels
        cache = kernels.Kv8Cache(state["k"], state["v"], state["sk"], state["sv"], state["table"])
        if kind == "append":
            kernels.kv8_append(state["new_k"], state["new_v"], cache, state["place"], layer=0, seq=state["seq"], rope_pos=state["pos"],
                               rope_cos=state["cos"], rope_sin=state["sin"], weight=state["weight"], position=state["position"])
            return {n: state[n] for n in ("k", "v", "sk", "sv", "weight", "position")}
        if kind == "tree":
            out, lse = kernels.attention_tree(state["q"], cache, state["start"], layer=0, n_q=case["n_q"], nodes=case["nodes"], count=state["count"], mask=state["mask"],
                                              rope_pos=state["pos"], rope_cos=state["cos"], rope_sin=state["sin"], max_len=state["max_len"], want_lse=True)
            return {"out": out, "lse": lse}
        if kind == "weigh":
            kernels.kv8_weigh(state["q"], state["lse"], cache, state["weight"], state["start"], layer=0, n_q=case["n_q"], nodes=case["nodes"], count=state["count"],
                              mask=state["mask"], rope_pos=state["pos"], rope_cos=state["cos"], rope_sin=state["sin"], max_len=state["max_len"])
            return {"weight": state["weight"]}
        if kind == "evict":
            length = kernels.kv8_evict(cache, state["weight"], state["position"], state["length"], keep=case["keep"], protect_from=state["from"], max_len=case["context"])
            return {"length": length} | {n: state[n] for n in ("k", "v", "sk", "sv", "weight", "position")}
        accepted, token, path = kernels.kv8_accept(cache, state["token"], state["parent"], state["chosen"], state["start"], count=state["count"],
                                                   weight=state["weight"], position=state["position"])
        return {"accepted": accepted, "next": token, "path": path} | {n: state[n] for n in ("k", "v", "sk", "sv", "weight", "position")}
    return {"append": _plain_append, "tree": _plain_tree, "weigh": _plain_weigh, "evict": _plain_evict, "accept": _plain_accept}[kind](state)


def _rotated(x, cos, sin):
    """x [rows, heads, 128] rotated as pairs (i, i + 64): one product rounded, the other fused with the sum."""
    a, b = x[..., :64], x[..., 64:]
    c, s = cos[:, None], sin[:, None]
    first = (a.double() * c.double() - (b * s).double()).float()
    second = (a.double() * s.double() + (b * c).double()).float()
    return torch.cat([first, second], -1)


def _plain_append(state):
    case, place, pos = state["case"], state["place"].long(), state["pos"].long()
    n_kv, slots = case["n_kv"], case["slots"]
    there = place >= 0
    at = place.clamp(min=0)
    rows = torch.stack([_rotated(state["new_k"].unflatten(-1, (n_kv, HD)), state["cos"][pos], state["sin"][pos]), state["new_v"].unflatten(-1, (n_kv, HD))])
    scale = rows.abs().amax(-1).clamp(min=1e-8) / 127.0
    code = (rows * scale.reciprocal()[..., None]).double()
    code = (code.abs() + 0.5).floor().copysign(code).clamp(-128, 127).to(torch.int8)      # halves away from zero
    block, slot = state["table"][state["seq"].long(), at // slots].long(), at % slots
    # a padding row is given the place of the row in front of it, and that row's contents
    source = torch.where(there, torch.arange(len(place), device=place.device), 0).cummax(0).values
    where = block[source], slot[source]
    for i, (rows_of, scales_of) in enumerate((("k", "sk"), ("v", "sv"))):
        state[rows_of][:, 0].transpose(1, 2)[where] = code[i][source]
        state[scales_of][:, 0].transpose(1, 2)[where] = scale[i][source]
    state["weight"][:, 0].transpose(1, 2)[where] = 0.0
    state["position"][:, 0].transpose(1, 2)[where] = state["pos"][source][:, None]
    return {n: state[n] for n in ("k", "v", "sk", "sv", "weight", "position")}


def _of_sequences(pool, table):
    """[sequences, heads, places(, 128)] of a cache's layer 0."""
    x = pool[:, 0][table.long()]                                    # [sequences, columns, heads, slots(, 128)]
    return x.transpose(1, 2).flatten(2, 3)


def _scores(state):
    """softmax's arguments [sequences, kv heads, nodes * heads of one, places], -inf where a node sees no key, and their log-sum-exp [rows, heads]."""
    case = state["case"]
    n_q, n_kv, nodes = case["n_q"], case["n_kv"], case["nodes"]
    sequences, group = case["sequences"], n_q // n_kv
    pos = state["pos"].long()
    q = _rotated(state["q"].unflatten(-1, (n_q, HD)), state["cos"][pos], state["sin"][pos])
    q = q.view(sequences, nodes, n_kv, group, HD).transpose(1, 2).flatten(2, 3)
    k = _of_sequences(state["k"], state["table"]).float() * _of_sequences(state["sk"], state["table"])[..., None]
    scores = (q @ k.transpose(-1, -2)) * (1.0 / math.sqrt(HD))
    node = torch.arange(k.shape[2], device=pos.device) - state["start"][:, None]                  # [sequences, places]
    inside = node.clamp(0, nodes - 1)
    bits = (state["mask"].view(sequences, nodes, -1).gather(2, (inside // 32).long()[:, None].expand(-1, nodes, -1)) >> (inside % 32)[:, None]) & 1
    seen = (node < 0)[:, None] | ((node >= 0) & (node < state["count"][:, None]))[:, None] & (bits == 1)
    seen = seen & (torch.arange(nodes, device=pos.device) < state["count"][:, None])[:, :, None]    # [sequences, nodes, places]
    scores = scores.unflatten(2, (nodes, group)).masked_fill_(~seen[:, None, :, None], -torch.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-1e30)
    lse = (scores - top).exp().sum(-1, dtype=torch.float64).log() + top.squeeze(-1).double()       # [sequences, kv heads, nodes, group]
    return scores, lse.float().transpose(1, 2).reshape(sequences * nodes, n_q)


def _weights(scores, lse, case):
    lse = lse.view(case["sequences"], case["nodes"], case["n_kv"], -1, 1).transpose(1, 2)
    return torch.where(torch.isfinite(lse), (scores - lse).exp(), 0.0)


def _plain_tree(state):
    case = state["case"]
    scores, lse = _scores(state)
    top = scores.amax(-1, keepdim=True).clamp(min=-1e30)
    w = scores.sub_(top).exp_()
    total = w.sum(-1, keepdim=True)
    v = _of_sequences(state["v"], state["table"]).float() * _of_sequences(state["sv"], state["table"])[..., None]
    out = (w.flatten(2, 3) @ v).unflatten(2, (case["nodes"], -1))
    out = torch.where(total > 0, out / total, 0.0)
    return {"out": out.transpose(1, 2).reshape(-1, case["n_q"] * HD), "lse": lse}


def _plain_weigh(state):
    case, table, slots = state["case"], state["table"], state["case"]["slots"]
    scores, _ = _scores(state)
    added = _weights(scores, state["lse"], case).sum((2, 3))                                       # [sequences, kv heads, places]
    state["weight"][:, 0].index_add_(0, table.long().flatten(), added.unflatten(-1, (-1, slots)).transpose(1, 2).flatten(0, 1))
    return {"weight": state["weight"]}


def _rows_of(pool, table):
    """[sequences, layers, heads, places(, 128)] of the whole cache."""
    return pool[table.long()].movedim(1, 3).flatten(3, 4)


def _plain_evict(state):
    case, table, slots, keep = state["case"], state["table"], state["case"]["slots"], state["case"]["keep"]
    length = state["length"].long()
    weight = _rows_of(state["weight"], table)
    place = torch.arange(weight.shape[-1], device=weight.device).expand(weight.shape)
    held = place < length[:, None, None, None]
    late = _rows_of(state["position"], table) >= state["from"][:, None, None, None]
    rank = torch.where(late, torch.inf, weight).masked_fill(~held, -torch.inf).argsort(dim=-1, descending=True, stable=True)
    keeps = torch.zeros_like(held).scatter_(-1, rank[..., :keep], True) & held
    hole, far = ~keeps & (place < keep) & held, keeps & (place >= keep)
    # the n-th token that is kept behind the budget goes to the n-th place that became free within it
    nth = lambda m: torch.where(m, m.long().cumsum(-1) - 1, m.shape[-1])                            # noqa: E731
    source = torch.zeros(*place.shape[:-1], place.shape[-1] + 1, dtype=torch.long, device=place.device)
    source = source.scatter_(-1, nth(far), place)[..., :-1].gather(-1, nth(hole).clamp(max=place.shape[-1] - 1))
    s, la, h, t = torch.nonzero(hole, as_tuple=True)
    f = source[s, la, h, t]
    old, new = (table[s, f // slots].long(), la, h, f % slots), (table[s, t // slots].long(), la, h, t % slots)
    for name in ("k", "v", "sk", "sv", "weight", "position"):
        state[name][new] = state[name][old]
    return {"length": state["length"].clamp(max=keep)} | {n: state[n] for n in ("k", "v", "sk", "sv", "weight", "position")}


def _plain_accept(state):
    case, table, slots = state["case"], state["table"], state["case"]["slots"]
    token, parent, chosen = state["token"], state["parent"].long(), state["chosen"]
    n = token.shape[1]
    node = torch.arange(n, device=token.device)
    from_node = parent.clamp(min=0)
    fits = (parent >= 0) & (parent < node) & (token == chosen.gather(1, from_node)) & (node < state["count"][:, None])
    first = ~((parent[:, :, None] == parent[:, None, :]) & fits[:, None, :] & (node[None, :] < node[:, None])).any(-1)
    on = (fits & first) | ((node == 0) & (state["count"][:, None] > 0))
    up = torch.where(node == 0, 0, from_node)
    for _ in range(max(1, n - 1).bit_length()):                                                   # a node counts if all in front of it do
        on, up = on & on.gather(1, up), up.gather(1, up)
    accepted = on.sum(1)
    rank = torch.where(on, on.long().cumsum(1) - 1, n)
    path = torch.full((len(token), n + 1), -1, dtype=torch.int32, device=token.device).scatter_(1, rank, node.to(torch.int32).expand(len(token), n))[:, :n]
    path = torch.where(node < accepted[:, None], path, -1)
    last = path.gather(1, (accepted - 1).clamp(min=0)[:, None]).long().clamp(min=0)
    following = torch.where(accepted > 0, chosen.gather(1, last).squeeze(1), -1)
    s, d = torch.nonzero(path >= 0, as_tuple=True)
    f, t = state["start"].long()[s] + path[s, d], state["start"].long()[s] + d
    old, new = (table[s, f // slots].long(), f % slots), (table[s, t // slots].long(), t % slots)
    for name in ("k", "v", "sk", "sv", "weight", "position"):
        rows = state[name].movedim(3, 1)
        rows[new] = rows[old]
    return {"accepted": accepted.to(torch.int32), "next": following, "path": path} | {n: state[n] for n in ("k", "v", "sk", "sv", "weight", "position")}


# ---- 64 bits -----------------------------------------------------------------------------------------------------------
def _exact_append(s, case):
    """The scales of the stored rows; the codes are whole numbers."""
    out = {"sk": s["sk"].double().cpu().numpy(), "sv": s["sv"].double().cpu().numpy()}
    place, seq, pos, table = (s[n].cpu().numpy() for n in ("place", "seq", "pos", "table"))
    real = np.flatnonzero(place >= 0)
    c, sn = (s[n].double().cpu().numpy()[pos[real]][:, None] for n in ("cos", "sin"))
    blocks, slots = table[seq[real], place[real] // case["slots"]], place[real] % case["slots"]
    for name, new in (("sk", "new_k"), ("sv", "new_v")):
        x = s[new].double().cpu().numpy()[real].reshape(len(real), case["n_kv"], 2, 64)
        if name == "sk":
            x = np.stack([x[:, :, 0] * c - x[:, :, 1] * sn, x[:, :, 0] * sn + x[:, :, 1] * c], 2)
        out[name][blocks, 0, :, slots] = np.maximum(np.abs(x).max((2, 3)), 1e-8) / 127
    weight = s["weight"].double().cpu().numpy()
    weight[blocks, 0, :, slots] = 0
    return {"k": None, "v": None, "sk": torch.from_numpy(out["sk"]), "sv": torch.from_numpy(out["sv"]), "weight": torch.from_numpy(weight), "position": None}


def _exact_attention(s, case):
    """Per sequence, kv head and node: (sequence, kv head, node, arguments [group, keys], keys' places), node after node from its line back to the root."""
    group, n_kv, slots = case["n_q"] // case["n_kv"], case["n_kv"], case["slots"]
    pos, half = s["pos"].cpu().numpy(), HD // 2
    for i, (start, count) in enumerate(zip(_starts(case), _counts(case))):
        line = []
        for j, p in enumerate(_parents(count, i)):
            line.append((line[p] if p >= 0 else []) + [j])
        places = torch.arange(start + count, device="cuda")
        blocks, at = s["table"][i].long()[places // slots], places % slots
        key = s["k"][blocks, 0, :, at].double() * s["sk"][blocks, 0, :, at].double()[..., None]     # [places, heads, 128]
        value = s["v"][blocks, 0, :, at].double() * s["sv"][blocks, 0, :, at].double()[..., None]
        r = torch.arange(count, device="cuda") + i * case["nodes"]
        turn = torch.from_numpy(pos[i * case["nodes"]: i * case["nodes"] + count].astype(np.int64)).cuda()
        c, sn = s["cos"][turn].double()[:, None, None], s["sin"][turn].double()[:, None, None]
        x = s["q"][r].double().view(count, n_kv, group, 2, half)
        x = torch.stack([x[..., 0, :] * c - x[..., 1, :] * sn, x[..., 0, :] * sn + x[..., 1, :] * c], -2).reshape(count, n_kv, group, HD)
        seen = torch.zeros(count, start + count, dtype=torch.bool, device="cuda")
        seen[:, :start] = True
        a, b = zip(*[(j, start + k) for j, ks in enumerate(line) for k in ks])
        seen[list(a), list(b)] = True
        for h in range(n_kv):
            score = torch.einsum("ngd,td->ngt", x[:, h], key[:, h]) / math.sqrt(HD)
            yield i, h, score.masked_fill(~seen[:, None], -math.inf), value[:, h], blocks, at


def _exact_tree(s, case):
    rows, n_q, n_kv = case["sequences"] * case["nodes"], case["n_q"], case["n_kv"]
    out = torch.zeros(rows, n_kv, n_q // n_kv, HD, dtype=torch.float64, device="cuda")
    lse = torch.full((rows, n_kv, n_q // n_kv), -math.inf, dtype=torch.float64, device="cuda")
    for i, h, score, value, _, _ in _exact_attention(s, case):
        r = slice(i * case["nodes"], i * case["nodes"] + score.shape[0])
        out[r, h] = torch.einsum("ngt,td->ngd", torch.softmax(score, -1), value)
        lse[r, h] = torch.logsumexp(score, -1)
    return {"out": out.view(rows, -1), "lse": lse.view(rows, n_q)}


def _exact_weigh(s, case):
    weight = s["weight"].double()
    lse = s["lse"].double().view(case["sequences"], case["nodes"], case["n_kv"], -1)
    for i, h, score, _, blocks, at in _exact_attention(s, case):
        weight[blocks, 0, h, at] += torch.exp(score - lse[i, : score.shape[0], h][..., None]).sum((0, 1))
    return {"weight": weight}


def exact(case, seed):
    if case["kind"] in ("evict", "accept"):     # rows are moved, nothing is computed
        return None
    s = prepare(case, seed)
    return {"append": _exact_append, "tree": _exact_tree, "weigh": _exact_weigh}[case["kind"]](s, case)
