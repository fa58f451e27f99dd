"""Plain 64-bit forms of the paged-cache operators (numpy), and batches of sequences over pages."""
import numpy as np

F32, F16, Q4_0, BF16 = 0, 1, 2, 30
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def norm_rope(x, w, eps, table, positions, dims, neox):
    """x [n, heads, dim]: heads normed by w (None: not), their first dims values rotated (table None: not), in 64 bits."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * w.astype(np.float64)
    if table is None:
        return x
    cs = table.astype(np.float64)[positions][:, None]
    i = np.arange(dims // 2)
    a, b = (i, i + dims // 2) if neox == 1 else (2 * i, 2 * i + 1)
    y = x.copy()
    y[..., a] = x[..., a] * cs[..., 0] - x[..., b] * cs[..., 1]
    y[..., b] = x[..., a] * cs[..., 1] + x[..., b] * cs[..., 0]
    return y


def rope_table(positions, dims, base=1e4):
    a = np.arange(positions)[:, None] * base ** (-np.arange(0, dims, 2) / dims)
    return np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)


def held(x, kind):
    """What a cache of this type stands for after rows x [..., dim] (rounded to 32 bits first), and for 4-bit rows how far
    each value is from the nearest border of its code, in codes (None for 16 bits)."""
    with np.errstate(all="ignore"):
        x = x.astype(np.float32)
        if kind == F16:
            return x.astype(np.float16).astype(np.float64), None
        b = x.reshape(-1, 32)
        fine = np.isfinite(b).all(1)
        size = np.abs(np.where(np.isfinite(b), b, 0))
        top = b[np.arange(len(b)), size.argmax(1)]
        d = (top * np.float32(-0.125)).astype(np.float16).astype(np.float64)
        fine &= np.abs(d) <= 8188
        u = b.astype(np.float64) / np.where(d == 0, 1, d)[:, None] + 8.5
        code = np.clip(np.floor(u), 0, 15)
        code[d == 0] = 8
        near = np.abs(u - np.round(u))
        near[(u < 0.5) | (u > 15.5)] = 1
        v = (code - 8) * d[:, None]
        v[~fine] = np.nan
        return v.reshape(x.shape), near.reshape(x.shape)


def attend(q, k, v, positions, held_at, scale, window):
    """One sequence: q [rows, heads, dim], k and v [length, kv_heads, dim] in 64 bits, the rows' positions, and which cached
    positions there are.  Returns the outputs, sum p |v|, the largest sum |q| |k| scale of each row's head, sum |v|, and the
    largest root of sum (q k scale)^2."""
    rows, heads, dim = q.shape
    group = heads // k.shape[1]
    t = np.arange(k.shape[0])
    out, mass, size, total, spread = (np.zeros((rows, heads, n)) for n in (dim, dim, 1, dim, 1))
    for r in range(rows):
        see = held_at & (t <= positions[r])
        if window:
            see &= t > positions[r] - window
        if not see.any():
            continue
        for h in range(heads):
            with np.errstate(all="ignore"):
                kk, vv = k[see, h // group], v[see, h // group]
                s = (kk @ q[r, h]) * scale
                if (s == -np.inf).all():
                    continue
                p = np.exp(s - s.max())
                p /= p.sum()
                out[r, h] = (p[:, None] * vv).sum(0)
                mass[r, h] = (p[:, None] * np.abs(vv)).sum(0)
                total[r, h] = np.abs(vv).sum(0)
                spread[r, h] = np.sqrt(((kk * q[r, h]) ** 2).sum(1).max()) * abs(scale)
                size[r, h] = (np.abs(kk) @ np.abs(q[r, h])).max() * abs(scale)
    return out, mass, size, total, spread


class Batch:
    """Sequences of given rows and lengths over shuffled pages of a pool."""

    def __init__(self, rows, lengths, page, seed=0, spare=2, pool=None):
        rng = np.random.default_rng(seed)
        self.rows, self.lengths, self.page = list(rows), list(lengths), page
        need = [-(-max(l, 0) // page) for l in lengths]
        self.pages = pool or sum(need) + spare
        self.stride = max(max(need), 1) + 1
        self.table = np.full((len(rows), self.stride), -1, np.int32)
        order = rng.permutation(self.pages).astype(np.int32)
        if pool:
            order = order[::-1]
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.free = order[at:]
        self.starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.n = int(self.starts[-1])

    def positions(self):
        return np.concatenate([np.arange(l - r, l) for r, l in zip(self.rows, self.lengths)] + [np.zeros(0, int)]).astype(np.int64)
