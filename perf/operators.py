"""Operators of beam search over a paged cache of 4-bit keys and values: appending and reading rows, decode attention, the
selection of continuations, and the forking of the cache to the selected beams.

A cached row (one token, one kv head, keys or values) is 80 bytes: 64 bytes of codes (dim d in nibble d % 2 of byte d / 2, the
low one first) and four pairs (scale, minimum) of fp16 for the dims 32g .. 32g + 31; a value is minimum + scale * code. The pool is
uint8 [block][layer][kv head][K, V][16 slots][80]; token t of a sequence lies in block block_table[sequence][t / 16], slot t % 16.

`own` says which side run() takes: the operators in elementary torch operations, or the framework's kernels.
"""
import math

import numpy as np
import torch

own = False

SLOTS, ROW, HD = 16, 80, 128
FP16_MOST = 65504.0


def listed():
    return [
        # The cache half of a decode step: one new token for each of 64 sequences.
        {"name": "append_step_64", "kind": "append", "sequences": 64, "tokens": 1, "n_kv": 5, "context": 1500, "padded": False},
        # A page of text and a batch of ragged prompts, some rows of the batch being padding.
        {"name": "append_prompt_1537", "kind": "append", "sequences": 1, "tokens": 1537, "n_kv": 5, "context": 0, "padded": False},
        {"name": "append_ragged_8x1000", "kind": "append", "sequences": 8, "tokens": 1000, "n_kv": 8, "context": 333, "padded": True},
        # One conversation, then one with four beams deep into a long text.
        {"name": "attention_1x1000", "kind": "attention", "sequences": 1, "rows": 1, "context": 1000, "ragged": False, "n_q": 20, "n_kv": 5},
        {"name": "attention_4x16000", "kind": "attention", "sequences": 4, "rows": 1, "context": 16001, "ragged": False, "n_q": 32, "n_kv": 8},
        # A server's decode step of one layer: equal lengths, and 256 ragged ones.
        {"name": "attention_64x8192", "kind": "attention", "sequences": 64, "rows": 1, "context": 8192, "ragged": False, "n_q": 20, "n_kv": 5},
        {"name": "attention_256_ragged", "kind": "attention", "sequences": 256, "rows": 1, "context": 4095, "ragged": True, "n_q": 20, "n_kv": 5},
        # A step of beam search: one request with four beams, a batch of 32 with eight, an odd vocabulary with many candidates.
        {"name": "select_1x4", "kind": "select", "groups": 1, "beams": 4, "vocab": 128256, "k": 8},
        {"name": "select_32x8", "kind": "select", "groups": 32, "beams": 8, "vocab": 128256, "k": 16},
        {"name": "select_5x12_odd", "kind": "select", "groups": 5, "beams": 12, "vocab": 50001, "k": 24},
        # The beams of one request, and of 64, take over their parents' caches in all 30 layers.
        {"name": "reorder_1x4", "kind": "reorder", "groups": 1, "beams": 4, "layers": 30, "n_kv": 5, "context": 219},
        {"name": "reorder_64x8", "kind": "reorder", "groups": 64, "beams": 8, "layers": 30, "n_kv": 5, "context": 1500},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "select", "reorder"])
    if kind == "append":
        sequences = _log_int(rng, 1, 256)
        tokens = _log_int(rng, 1, max(1, 8000 // sequences))
        return {"kind": kind, "sequences": sequences, "tokens": tokens, "n_kv": rng.choice([1, 2, 5, 5, 8, 16] if sequences * tokens < 4000 else [1, 5, 8]),
                "context": _log_int(rng, 1, 2000) - 1, "padded": rng.random() < 0.5}
    if kind == "attention":
        n_q, n_kv = rng.choice([(20, 5), (20, 5), (32, 8), (16, 16), (40, 5), (12, 4), (7, 1), (32, 2), (6, 1)])
        rows = rng.choice([1, 1, 1, 2, 5])
        sequences = _log_int(rng, 1, 256)
        context = min(_log_int(rng, rows, 16384), 2600000 // (sequences * rows * n_kv))
        return {"kind": kind, "sequences": sequences, "rows": rows, "context": max(rows, context), "ragged": rng.random() < 0.7, "n_q": n_q, "n_kv": n_kv}
    if kind == "select":
        beams = rng.randint(1, 16)
        vocab = rng.choice([128256, 1024, _log_int(rng, 500, 128256)])
        groups = min(_log_int(rng, 1, 64), max(1, 32 * 8 * 128256 // (beams * vocab)))
        return {"kind": kind, "groups": groups, "beams": beams, "vocab": vocab, "k": rng.choice([beams, 2 * beams])}
    beams = rng.randint(2, 16)
    n_kv, layers = rng.choice([(5, 30), (8, 32), (1, 2)])
    return {"kind": kind, "groups": _log_int(rng, 1, 64 * 8 // beams), "beams": beams, "layers": layers if n_kv < 8 else rng.choice([8, 16]), "n_kv": n_kv,
            "context": _log_int(rng, 1, 2000)}


# ---- sizes -------------------------------------------------------------------------------------------------------------
def _spread(most, count, least=1):
    """Lengths of a batch: from half of `most` to `most`, as in a server that admits requests one by one."""
    return [max(least, most - (i * 2654435761 >> 7) % max(1, most // 2)) for i in range(count)]


def _append_rows(case):
    """(sequence, position) of each row; position -1 where the row is padding."""
    rows = []
    for s in range(case["sequences"]):
        start = case["context"] - (s * 40503) % max(1, case["context"] // 2 + 1)
        real = case["tokens"] - (s * 97) % max(1, case["tokens"] // 3 + 1) if case["padded"] else case["tokens"]
        rows += [(s, start + i if i < real else -1) for i in range(case["tokens"])]
    return rows


def _attention_rows(case):
    """(sequence, position) of each query row: the last `rows` tokens of every sequence."""
    lengths = _spread(case["context"], case["sequences"], case["rows"]) if case["ragged"] else [case["context"]] * case["sequences"]
    return [(s, n - case["rows"] + r) for s, n in enumerate(lengths) for r in range(case["rows"])]


def work(case):
    kind = case["kind"]
    if kind == "append":            # fp32 rows in, their 160 bytes a head out, and the same back as fp32
        rows = _append_rows(case)
        real = sum(p >= 0 for _, p in rows)
        values = 2 * HD * case["n_kv"]
        return {"bytes": real * (4 * values + 2 * ROW * case["n_kv"]) * 2 + 8 * len(rows), "flops": 12 * real * values}
    if kind == "attention":
        rows = _attention_rows(case)
        cached = sum(p + 1 for _, p in rows[case["rows"] - 1:: case["rows"]])
        scored = sum(p + 1 for _, p in rows)
        return {"bytes": cached * (2 * ROW * case["n_kv"] + 4 / SLOTS) + 2 * len(rows) * case["n_q"] * HD * 4, "flops": 4 * scored * case["n_q"] * HD}
    if kind == "select":
        n = case["groups"] * case["beams"] * case["vocab"]
        return {"bytes": 4 * n + 12 * case["groups"] * case["k"], "flops": 3 * n}
    b, g = case["beams"], case["groups"]
    copied = b * (1 - 1 / b) ** b   # beams that no other continues, each of which takes a copy
    tail = sum(n % SLOTS for n in _spread(case["context"], g)) * 2 * ROW * case["n_kv"] * case["layers"]
    return {"bytes": 2 * copied * tail + 8 * g * b * _blocks(case["context"] + 1), "flops": 0}


# ---- states ------------------------------------------------------------------------------------------------------------
def _blocks(tokens):
    return (tokens + SLOTS - 1) // SLOTS


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _pool(g, blocks, layers, n_kv):
    """Rows as quantising values near N(0, 1) leaves them: codes thickest in the middle, groups of their own scale and minimum."""
    pool = torch.empty(blocks, layers, n_kv, 2, SLOTS, ROW, dtype=torch.uint8, device="cuda")
    shape = (blocks, layers, n_kv, 2, SLOTS, HD // 2)
    pool[..., :64] = torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8).bitwise_and_(0x77)
    pool[..., :64] += torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8).bitwise_and_(0x77)
    params = torch.empty(shape[:-1] + (4, 2), dtype=torch.float16, device="cuda")
    params[..., 0] = 0.2 + 0.15 * torch.rand(shape[:-1] + (4,), generator=g, device="cuda")
    params[..., 1] = -params[..., 0] * (6.5 + torch.rand(shape[:-1] + (4,), generator=g, device="cuda"))
    pool[..., 64:] = params.flatten(-2).view(torch.uint8)
    return pool


def _table(g, sequences, columns):
    """Every sequence has blocks of its own, from anywhere in the pool."""
    return torch.randperm(sequences * columns, generator=g, device="cuda").to(torch.int32).view(sequences, columns)


def _rope(length):
    at = torch.arange(length, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-torch.arange(64, dtype=torch.float64, device="cuda") / 64)
    return at.cos().float(), at.sin().float()


def prepare(case, seed):
    g, kind = _generator(seed), case["kind"]
    s = {"case": case}
    if kind in ("append", "attention"):
        rows = _append_rows(case) if kind == "append" else _attention_rows(case)
        s["pos"] = torch.tensor([p for _, p in rows], dtype=torch.int32, device="cuda")
        s["seq"] = torch.tensor([q for q, _ in rows], dtype=torch.int32, device="cuda")
        most = max(p for _, p in rows) + 1
        s["max_len"], columns = most, _blocks(most)
        s["table"] = _table(g, case["sequences"], columns)
        s["cos"], s["sin"] = _rope(most)
        s["pool"] = _pool(g, case["sequences"] * columns, 1, case["n_kv"])
        if kind == "append":
            for name in ("k", "v"):     # values of a projection: some dims a good deal larger than the rest
                s[name] = torch.randn(len(rows), case["n_kv"] * HD, generator=g, device="cuda")
                s[name] *= torch.exp(0.7 * torch.randn(case["n_kv"] * HD, generator=g, device="cuda"))
        else:
            s["q"] = 1.5 * torch.randn(len(rows), case["n_q"] * HD, generator=g, device="cuda")
        return s
    if kind == "select":
        rows = case["groups"] * case["beams"]
        s["logits"] = 2.5 * torch.randn(rows, case["vocab"], generator=g, device="cuda")
        s["logits"][:, 7: case["vocab"]: 911] = -torch.inf      # tokens that are not allowed
        s["scores"] = -20.0 - 2.0 * torch.rand(rows, generator=g, device="cuda")
        s["finished"] = (torch.rand(rows, generator=g, device="cuda") < 0.1).to(torch.int32)
        return s
    groups, beams, columns = case["groups"], case["beams"], _blocks(case["context"] + 1)
    s["length"] = torch.tensor(_spread(case["context"], groups), dtype=torch.int32, device="cuda")
    s["parent"] = torch.randint(0, beams, (groups, beams), generator=g, device="cuda", dtype=torch.int32)
    blocks = groups * beams * 2                                  # the blocks that are being filled, and as many full ones
    s["table"] = torch.randint(0, blocks // 2, (groups * beams, columns), generator=g, device="cuda", dtype=torch.int32)
    tails = blocks // 2 + torch.randperm(blocks // 2, generator=g, device="cuda").to(torch.int32)
    at = (s["length"] // SLOTS).repeat_interleave(beams).long()
    s["table"].scatter_(1, at[:, None], tails[:, None])
    s["pool"] = torch.randint(-2 ** 31, 2 ** 31 - 1, (blocks, case["layers"], case["n_kv"], 2, SLOTS, ROW // 4), generator=g, device="cuda", dtype=torch.int32)
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------------
EOS = 2


def run(state):
    kind, case = state["case"]["kind"], state["case"]
    if own:
        from tenzo_b200 import kernels
        if kind == "append":
            kernels.kv4_append(state["k"], state["v"], state["pool"], state["pos"], layer=0, block_table=state["table"], seq=state["seq"],
                               rope_cos=state["cos"], rope_sin=state["sin"])
            k, v = kernels.kv4_read(state["pool"], state["pos"], layer=0, block_table=state["table"], seq=state["seq"])
            return {"k": k, "v": v}
        if kind == "attention":
            return kernels.attention_kv4(state["q"], state["pool"], state["pos"], layer=0, n_q=case["n_q"], block_table=state["table"], seq=state["seq"],
                                         rope_cos=state["cos"], rope_sin=state["sin"], max_len=state["max_len"])
        if kind == "select":
            parent, token, score = kernels.beam_select(state["logits"], state["scores"], beams=case["beams"], k=case["k"], finished=state["finished"], eos=EOS)
            return {"parent": parent, "token": token, "score": score}
        table = kernels.kv4_reorder(state["pool"].view(torch.uint8), state["table"], state["parent"], state["length"])
        return {"table": table, "pool": state["pool"]}
    if kind == "append":
        return _plain_append(state)
    if kind == "attention":
        return _plain_attention(state)
    return _plain_select(state) if kind == "select" else _plain_reorder(state)


def _rotated(x, cos, sin):
    """x [rows, heads, 128] rotated as pairs (i, i + 64): one product rounded, the other fused with the sum."""
    a, b = x[..., :64], x[..., 64:]
    c, s = cos[:, None], sin[:, None]
    first = (a.double() * c.double() - (b * s).double()).float()
    second = (a.double() * s.double() + (b * c).double()).float()
    return torch.cat([first, second], -1)


def _quantised(x):
    """Rows [..., 128] as 80 bytes each, every step rounded to fp32 (the parameters to fp16)."""
    x = x.clamp(-FP16_MOST, FP16_MOST).unflatten(-1, (4, 32))
    low = x.amin(-1, keepdim=True).half()
    scale = ((x.amax(-1, keepdim=True) - low.float()) * (1.0 / 15)).half()
    code = ((x - low.float()) * scale.float().reciprocal()).round().clamp(0, 15)
    code = torch.where(scale > 0, code, torch.zeros_like(code)).to(torch.uint8).flatten(-2)
    return torch.cat([code[..., 0::2] | code[..., 1::2] << 4, torch.cat([scale, low], -1).flatten(-2).contiguous().view(torch.uint8)], -1)


def _values(rows):
    """The fp32 values of rows [..., 80]."""
    params = rows[..., 64:].contiguous().view(torch.float16).float().unflatten(-1, (4, 2))
    code = torch.stack([rows[..., :64] & 15, rows[..., :64] >> 4], -1).flatten(-2).float().unflatten(-1, (4, 32))
    return (code * params[..., 0:1] + params[..., 1:2]).flatten(-2)


def _plain_append(state):
    pos, pool = state["pos"].long(), state["pool"]
    there = pos >= 0
    at = pos.clamp(min=0)
    n_kv = pool.shape[2]
    k = _rotated(state["k"].unflatten(-1, (n_kv, HD)), state["cos"][at], state["sin"][at])
    new = _quantised(torch.stack([k, state["v"].unflatten(-1, (n_kv, HD))], 2))
    block, slot = state["table"][state["seq"].long(), at // SLOTS].long(), at % SLOTS
    keep = there[:, None, None, None]
    # a padding row is given the place of the row in front of it, and that row's contents
    source = torch.where(there, torch.arange(len(pos), device=pos.device), 0).cummax(0).values
    pool[:, 0].transpose(1, 3)[block[source], slot[source]] = new.transpose(1, 2)[source]
    back = _values(pool[:, 0].transpose(1, 3)[block, slot])         # [rows, K|V, heads, 128]
    back = torch.where(keep, back, torch.zeros_like(back))
    return {"k": back[:, 0].flatten(1), "v": back[:, 1].flatten(1)}


def _plain_attention(state):
    case, pos, pool = state["case"], state["pos"].long(), state["pool"]
    n_kv, group = case["n_kv"], case["n_q"] // case["n_kv"]
    q = _rotated(state["q"].unflatten(-1, (case["n_q"], HD)), state["cos"][pos], state["sin"][pos]).unflatten(1, (n_kv, group))
    pages = pool[:, 0][state["table"][state["seq"].long()].long()]  # [rows, blocks, heads, K|V, slots, 80]
    kv = _values(pages.permute(3, 0, 2, 1, 4, 5).flatten(3, 4))     # [K|V, rows, heads, tokens, 128]
    scores = (q @ kv[0].transpose(-1, -2)) * (1.0 / math.sqrt(HD))
    seen = torch.arange(scores.shape[-1], device=pos.device) <= pos[:, None, None, None]
    scores = torch.where(seen, scores, torch.full_like(scores, -torch.inf))
    weights = (scores - scores.amax(-1, keepdim=True)).exp()
    return ((weights @ kv[1]) / weights.sum(-1, keepdim=True)).flatten(1)


def _plain_select(state):
    case = state["case"]
    x = state["logits"].double()
    m = x.amax(-1, keepdim=True)
    logsum = m + (x - m).exp().sum(-1, keepdim=True).log()
    scores = state["scores"].double()[:, None] + (x - logsum)
    done = state["finished"][:, None] != 0
    only = torch.where(torch.arange(case["vocab"], device=x.device) == EOS, state["scores"].double()[:, None], -torch.inf)
    scores = torch.where(done, only, scores).view(case["groups"], -1)
    best, at = torch.sort(scores, dim=-1, descending=True, stable=True)
    at = at[:, : case["k"]]
    return {"parent": (at // case["vocab"]).to(torch.int32), "token": (at % case["vocab"]).to(torch.int32), "score": best[:, : case["k"]].float()}


def _plain_reorder(state):
    case, table, pool, parent = state["case"], state["table"], state["pool"], state["parent"].long()
    groups, beams = parent.shape
    columns = table.shape[1]
    old = table.view(groups, beams, columns)
    ids = torch.arange(beams, device=table.device)
    same = parent[:, :, None] == parent[:, None, :]                       # [group, child, other child]
    further = (same & (ids[None, :] < ids[:, None])).any(-1)              # a child whose parent has one of a lower index
    childless = ~(parent[:, :, None] == ids).any(1)
    donors = torch.argsort((~childless).to(torch.int8), dim=-1, stable=True)  # childless beams first, by index
    nth = (further.long().cumsum(-1) - 1).clamp(min=0)
    giver = torch.where(further, donors.gather(1, nth), parent)           # whose tail block the child takes
    length = state["length"].long()
    column, filled = (length // SLOTS)[:, None], length % SLOTS
    tails = old.gather(2, column[:, :, None].expand(groups, beams, 1)).squeeze(2)
    x = torch.arange(columns, device=table.device)
    inherited = old.gather(1, parent[:, :, None].expand(groups, beams, columns))
    taken = torch.where(filled[:, None] > 0, tails.gather(1, giver), tails)
    new = torch.where(x < column[:, :, None], inherited, old)
    new = torch.where(x == column[:, :, None], taken[:, :, None], new)
    source, target = torch.where(filled[:, None] > 0, tails.gather(1, parent), tails).long().flatten(), taken.long().flatten()
    rows = (torch.arange(SLOTS, device=table.device) < filled[:, None]).repeat_interleave(beams, 0)[:, None, None, None, :, None]
    pool[target] = torch.where(rows, pool[source], pool[target])
    return {"table": new.view(groups * beams, columns), "pool": pool}


# ---- 64 bits -----------------------------------------------------------------------------------------------------------
def _decoded64(rows):
    """Rows [n, 80] (uint8) as 64-bit values [n, 128], nibble by nibble."""
    words = rows[:, :64].contiguous().view(torch.int32).to(torch.int64) & 0xFFFFFFFF
    shifts = 4 * torch.arange(8, device=rows.device)
    codes = ((words[:, :, None] >> shifts) & 15).reshape(len(rows), 4, 32).double()
    pairs = rows[:, 64:].contiguous().view(torch.float16).double().view(len(rows), 4, 2)
    return (pairs[:, :, 1, None] + codes * pairs[:, :, 0, None]).reshape(len(rows), HD)


def _exact_append(s, case):
    """The cached values by the quantiser's definition: its steps are fp32 by definition, so they are taken with numpy, one by one."""
    f = np.float32
    k, v = (s[n].cpu().numpy().reshape(-1, case["n_kv"], HD) for n in ("k", "v"))
    pos = s["pos"].cpu().numpy()
    at = np.maximum(pos, 0)
    cos, sin = s["cos"].cpu().numpy()[at][:, None], s["sin"].cpu().numpy()[at][:, None]
    lo, hi = k[..., :64], k[..., 64:]
    wide = np.float64
    k = np.concatenate([(lo.astype(wide) * cos.astype(wide) - (hi * sin).astype(wide)).astype(f),
                        (lo.astype(wide) * sin.astype(wide) + (hi * cos).astype(wide)).astype(f)], -1)
    out = {}
    for name, x in (("k", k), ("v", v)):
        x = np.clip(x, f(-FP16_MOST), f(FP16_MOST)).reshape(-1, 32)
        low = x.min(1).astype(np.float16)
        step = ((x.max(1) - low.astype(f)) * f(1.0 / 15)).astype(np.float16)
        with np.errstate(divide="ignore", invalid="ignore"):
            code = np.rint((x - low.astype(f)[:, None]) * (f(1) / step.astype(f))[:, None])
        code = np.where(step[:, None] > 0, np.clip(code, 0, 15), 0)
        value = low.astype(wide)[:, None] + step.astype(wide)[:, None] * code.astype(wide)
        value = value.reshape(len(pos), -1)
        value[pos < 0] = 0
        out[name] = torch.from_numpy(value)
    return out


def _exact_attention(s, case):
    group, out = case["n_q"] // case["n_kv"], []
    table, half = s["table"].cpu().numpy(), HD // 2
    for row, (q, p) in enumerate(zip(s["seq"].tolist(), s["pos"].tolist())):
        turn_c, turn_s = s["cos"][p].double(), s["sin"][p].double()
        x = s["q"][row].double().view(case["n_kv"], group, 2, half)
        x = torch.stack([x[:, :, 0] * turn_c - x[:, :, 1] * turn_s, x[:, :, 0] * turn_s + x[:, :, 1] * turn_c], 2).reshape(case["n_kv"], group, HD)
        blocks = torch.from_numpy(table[q, : _blocks(p + 1)].astype(np.int64)).cuda()
        page = s["pool"][blocks, 0]                                         # [blocks, heads, K|V, slots, 80]
        val = _decoded64(page.reshape(-1, ROW)).view(len(blocks), case["n_kv"], 2, SLOTS, HD)
        key, value = (val[:, :, i].permute(1, 0, 2, 3).reshape(case["n_kv"], -1, HD)[:, : p + 1] for i in (0, 1))
        w = torch.softmax(torch.bmm(x, key.transpose(1, 2)) / math.sqrt(HD), -1)
        out.append(torch.bmm(w, value).reshape(-1))
    return torch.stack(out)


def _exact_select(s, case):
    b, n, k = case["beams"], case["vocab"], case["k"]
    parents, tokens, scores = [], [], []
    before, done = s["scores"].double().cpu().numpy(), s["finished"].cpu().numpy()
    for g in range(case["groups"]):
        found = []
        for beam in range(b):
            r = g * b + beam
            x = s["logits"][r].cpu().numpy().astype(np.float64)
            if done[r]:
                x[:] = -np.inf
                x[EOS] = before[r]
            else:
                top = x.max()
                x = before[r] + (x - (top + np.log(np.sum(np.exp(x - top)))))
            border = np.partition(x, n - k)[n - k]
            found += [(-x[t], beam * n + t) for t in np.flatnonzero(x >= border)[: max(k, np.count_nonzero(x > border) + k)]] if border > -np.inf else \
                [(-x[t], beam * n + t) for t in np.argsort(-x, kind="stable")[:k]]
        found = sorted(found)[:k]
        parents.append([i // n for _, i in found])
        tokens.append([i % n for _, i in found])
        scores.append([-m for m, _ in found])
    return {"parent": torch.tensor(parents, dtype=torch.int32), "token": torch.tensor(tokens, dtype=torch.int32),
            "score": torch.tensor(np.array(scores), dtype=torch.float64)}


def exact(case, seed):
    if case["kind"] == "reorder":       # blocks are moved, nothing is computed
        return None
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "select": _exact_select}[case["kind"]](s, case)
