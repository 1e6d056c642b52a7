"""The 4-bit paged cache and beam selection in numpy, for the tests: the quantiser step by step in fp32 (its bits are a contract), everything
else in 64 bits."""
import numpy as np

F, D = np.float32, np.float64
SLOTS, ROW = 16, 80


def rope(length, theta=10000.0):
    at = np.arange(length)[:, None] * theta ** (-np.arange(64) / 64)
    return np.cos(at).astype(F), np.sin(at).astype(F)


def rotate(x, cos, sin):
    """x fp32 [..., 128], cos and sin fp32 [..., 64]: one product rounded, the other fused with the sum (exact in 64 bits, rounded once)."""
    a, b = x[..., :64], x[..., 64:]
    first = (a.astype(D) * cos - (b * sin).astype(D)).astype(F)
    second = (a.astype(D) * sin + (b * cos).astype(D)).astype(F)
    return np.concatenate([first, second], -1)


def quantise(x):
    """fp32 [..., 128] -> uint8 [..., 80]."""
    shape = x.shape[:-1]
    x = np.clip(x, F(-65504), F(65504)).reshape(-1, 4, 32)
    low = x.min(-1).astype(np.float16)
    scale = ((x.max(-1) - low.astype(F)) * F(1.0 / 15)).astype(np.float16)
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        code = np.rint((x - low.astype(F)[..., None]) * (F(1) / scale.astype(F))[..., None])
    code = np.where(scale[..., None] > 0, np.clip(code, 0, 15), 0).astype(np.uint8).reshape(-1, 128)
    rows = np.zeros((len(x), ROW), np.uint8)
    rows[:, :64] = code[:, 0::2] | code[:, 1::2] << 4
    rows[:, 64:] = np.stack([scale, low], -1).reshape(-1, 8).view(np.uint8)
    return rows.reshape(*shape, ROW)


def values(rows):
    """uint8 [..., 80] -> 64-bit [..., 128]."""
    code = np.stack([rows[..., :64] & 15, rows[..., :64] >> 4], -1).reshape(*rows.shape[:-1], 4, 32).astype(D)
    params = np.ascontiguousarray(rows[..., 64:]).view(np.float16).astype(D).reshape(*rows.shape[:-1], 4, 2)
    return (params[..., 1:] + params[..., :1] * code).reshape(*rows.shape[:-1], 128)


def cached(pool, layer, table_row, n):
    """The first n tokens of a sequence: (keys, values), 64-bit [n_kv, n, 128]."""
    blocks = table_row[: (n + SLOTS - 1) // SLOTS]
    v = values(pool[blocks, layer])                                      # [blocks, heads, 2, slots, 128]
    v = v.transpose(2, 1, 0, 3, 4).reshape(2, pool.shape[2], -1, 128)
    return v[0, :, :n], v[1, :, :n]


def attention(q, k, v, cos=None, sin=None):
    """q fp32 [n_q, 128] (before rotation), k and v 64-bit [n_kv, n, 128] -> (out [n_q, 128], bound): `bound` is how far an fp32 kernel with
    22-bit products may be off, element by element.

    The bound: a score is a sum of 128 products (and their parameters'), of which each and each partial sum is off by 2^-22 of the
    products' absolute sum at most where the rounding errors add up as random ones do, and 4 times that covers the worst row of a test;
    the exponential is off by 2^-21. A weight is then off by d = 2 * (4 * 2^-22 * mass) + 2^-20 relative, numerator and
    denominator alike, and the output by 2 d sum p|v|; |v| is taken as |minimum| + |scale * code| (at most 3 max|v|) because the kernel sums the two apart."""
    if cos is not None:
        c, s = cos.astype(D), sin.astype(D)
        a, b = q[:, :64].astype(D), q[:, 64:].astype(D)
        q = np.concatenate([a * c - b * s, a * s + b * c], -1)
    q = q.astype(D)
    n_q, n_kv, n = len(q), len(k), k.shape[1]
    if n == 0:
        return np.zeros((n_q, 128)), np.zeros((n_q, 128))
    k, v = np.repeat(k, n_q // n_kv, 0), np.repeat(v, n_q // n_kv, 0)
    s = np.einsum("hd,htd->ht", q, k) / np.sqrt(128.0)
    mass = np.einsum("hd,htd->ht", abs(q), abs(k)).max(-1, keepdims=True) / np.sqrt(128.0)
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    d = 2 * 4 * 2.0 ** -22 * mass + 2.0 ** -20
    spread = 3 * abs(v).reshape(n_q, n, 4, 32).max(-1).repeat(32, -1).reshape(n_q, n, 128)
    return np.einsum("ht,htd->hd", p, v), 2 * d * np.einsum("ht,htd->hd", p, spread) + 1e-30


def select(logits, scores, beams, k, finished=None, eos=0):
    """(parent, token, score) [groups, k]; score in 64 bits. Best score first; of equal ones the lower beam, in a beam the larger logit (tiny logits can
    differ and give the same 64-bit score), then the lower token."""
    x = logits.astype(D)
    x = np.where(np.isnan(x), -np.inf, np.minimum(x, D(np.finfo(F).max)))
    cum = np.where(np.isnan(scores), -np.inf, scores).astype(D)
    top = x.max(-1)
    with np.errstate(invalid="ignore", divide="ignore"):
        full = cum[:, None] + (x - (top + np.log(np.exp(x - top[:, None]).sum(-1)))[:, None])
    full[(top == -np.inf) | (cum == -np.inf)] = -np.inf
    if finished is not None:
        for r in np.flatnonzero(finished):
            full[r] = -np.inf
            full[r, eos] = cum[r]
    full, x = full.reshape(-1, beams * x.shape[1]), np.where(full == -np.inf, 0, x).reshape(-1, beams * x.shape[1])
    beam = np.arange(full.shape[1]) // logits.shape[1]
    at = np.stack([np.lexsort((-a, beam, -f))[:k] for a, f in zip(x, full)]) if len(full) else np.zeros((0, k), int)
    return at // logits.shape[1], at % logits.shape[1], np.take_along_axis(full, at, -1)


def reorder(pool, table, parent, length):
    """(new table, new pool)."""
    groups, beams = parent.shape
    new, pool = table.copy(), pool.copy()
    for g in range(groups):
        j, r = divmod(int(length[g]), SLOTS)
        rows, out = table[g * beams: (g + 1) * beams], new[g * beams: (g + 1) * beams]
        free = [b for b in range(beams) if b not in parent[g]]
        taken = set()
        for i, p in enumerate(parent[g]):
            out[i, :j] = rows[p, :j]
            if r == 0:
                continue
            if p not in taken:
                taken.add(p)
                out[i, j] = rows[p, j]
            else:
                out[i, j] = rows[free.pop(0), j]
                pool[out[i, j], :, :, :, :r] = pool[rows[p, j], :, :, :, :r]
    return new, pool


def random_pool(rng, blocks, layers, n_kv, spread=1.0):
    """Rows as the quantiser leaves values of N(0, spread^2)."""
    x = rng.standard_normal((blocks, layers, n_kv, 2, SLOTS, 128)).astype(F) * F(spread)
    return quantise(x)
