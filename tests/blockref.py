"""The block-scaled KV cache, the attention over it and log probabilities in float64 NumPy, from their definitions: what
the tests of t2r_amd.ops's block calls compare with."""
import numpy as np

F = np.float32
MAXF = np.finfo(F).max


class Cache:
    """The cache on the host, laid out as t2r_amd.ops.block_cache lays it out."""

    def __init__(self, n_blocks, Hk, hd, block):
        self.n, self.Hk, self.hd, self.bs = n_blocks, Hk, hd, block
        self.kc = np.zeros((n_blocks, Hk, block, hd), np.int8)
        self.vc = np.zeros((n_blocks, Hk, hd, block), np.int8)
        self.ks = np.zeros((n_blocks, Hk), F)
        self.vs = np.zeros((n_blocks, Hk), F)

    def places(self, table, starts, lens, rows):
        """(row, block or -1, slot, position) of every ragged row."""
        for b in range(len(lens)):
            n = starts[b + 1] - starts[b]
            for i in range(n):
                p = int(lens[b]) - n + i
                j = p // self.bs
                blk = int(table[b][j]) if 0 <= j < len(table[b]) else -1
                yield starts[b] + i, blk if 0 <= blk < self.n else -1, p % self.bs, p, b

    def append(self, k, v, table, starts, lens):
        groups = {}
        for r, blk, slot, p, b in self.places(table, starts, lens, len(k)):
            if blk >= 0:
                groups.setdefault(blk, []).append((r, slot))
        for blk, rs in groups.items():
            lo = min(s for _, s in rs)
            for x, code, scale in ((k, self.kc, self.ks), (v, self.vc.transpose(0, 1, 3, 2), self.vs)):
                y = np.asarray(x, np.float64).reshape(-1, self.Hk, self.hd)[[r for r, _ in rs]]
                y = np.clip(np.where(np.isnan(y), 0, y), -MAXF, MAXF)
                s = F(np.abs(y).max((0, 2)) / 127)                     # [Hk]
                old = scale[blk].copy() if lo else np.zeros(self.Hk, F)
                s = np.maximum(s, old)
                with np.errstate(invalid="ignore", divide="ignore"):
                    was = code[blk, :, :lo].astype(np.float64) * old.astype(np.float64)[:, None, None]
                    moved = np.nan_to_num(np.rint(was / s.astype(np.float64)[:, None, None]))
                    new = np.where(s[None, :, None] > 0, np.rint(y / s.astype(np.float64)[None, :, None]), 0)
                grew = (s > old) & (old > 0)
                code[blk, :, :lo] = np.where(grew[:, None, None], moved, code[blk, :, :lo])
                for (r, slot), q in zip(rs, np.clip(new, -127, 127)):
                    code[blk, :, slot] = q
                scale[blk] = s

    def values(self, table, b, n):
        """float64 keys and values [n, Hk, hd] of positions 0 .. n - 1 of sequence b, and whether each is there."""
        k, v, there = np.zeros((n, self.Hk, self.hd)), np.zeros((n, self.Hk, self.hd)), np.zeros(n, bool)
        for j in range(-(-n // self.bs)):
            blk = int(table[b][j]) if j < len(table[b]) else -1
            if not 0 <= blk < self.n:
                continue
            m = min(self.bs, n - j * self.bs)
            at = slice(j * self.bs, j * self.bs + m)
            k[at] = (self.kc[blk].astype(np.float64) * self.ks[blk].astype(np.float64)[:, None, None]).transpose(1, 0, 2)[:m]
            v[at] = (self.vc[blk].astype(np.float64) * self.vs[blk].astype(np.float64)[:, None, None]).transpose(2, 0, 1)[:m]
            there[at] = True
        return k, v, there


def attention(cache, q, table, starts, lens, H, scale, half=0.0, only=None):
    """(outputs [rows, H * hd], bound) in float64, of the rows `only` (default all; the others NaN); a row below position 0 is
    NaN, one that sees no position 0. bound: how far a float32 result may be off by the arithmetic that the
    kernels state. With A the largest sum |q_i k_i| scale of a row, n its keys and W the sum of p |v| for an element:
      - scores: q in two fp16 numbers 2^-22 relative (16-bit rows: nothing but 2^-25 of the row's largest value), sums of hd
        products (hd + 8) 2^-24: A (2^-22 + (hd + 8) 2^-24), and the same again in the denominator;
      - exp2 and its argument 2^-21 + A 2^-22, p vs / vref and its two fp16 pieces 2^-21, sums of n terms over 4 waves and 4
        lanes (n / 8 + 128) 2^-24;
      - p vs / vref is held with 2^11 put before the largest p, so fp16's last half step, 2^-25, is 2^-36 of it for each of n
        keys, times the largest value there is (vref is the largest scale of the keys at hand): n 2^-36 max |v|.
    `half`: 2^-11 where p is one fp16 number (16-bit rows)."""
    hd, Hk = cache.hd, cache.Hk
    q = np.asarray(q, np.float64).reshape(-1, H, hd)
    out, bound = np.zeros((len(q), H * hd)), np.zeros((len(q), H * hd))
    for b in range(len(lens)):
        n_new = starts[b + 1] - starts[b]
        if n_new == 0:
            continue
        most = max(int(lens[b]), 0)
        k, v, there = cache.values(table, b, most)
        for i in range(n_new):
            n = int(lens[b]) - n_new + i + 1
            if n < 0 or (n == 0 and n_new > 1) or (only is not None and starts[b] + i not in only):
                out[starts[b] + i] = np.nan
                continue
            ok = there[:n]
            if not ok.any():
                continue
            for h in range(H):
                kk, vv = k[:n, h * Hk // H][ok], v[:n, h * Hk // H][ok]
                x = q[starts[b] + i, h]
                s = kk @ x * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                A = (np.abs(kk) @ np.abs(x)).max() * scale
                tol = 2 * A * (2.0 ** -22 + (hd + 8) * 2.0 ** -24) + A * 2.0 ** -22 + 2.0 ** -20 + (n / 8 + 128) * 2.0 ** -24 + half
                at = (starts[b] + i, slice(h * hd, (h + 1) * hd))
                out[at] = p @ vv
                bound[at] = tol * (p @ np.abs(vv)) + n * 2.0 ** -36 * np.abs(v[:, h * Hk // H]).max()
    return out, bound


def logprobs(x, tokens, top):
    """(log p, entropy, ids, log p of the ids) in float64 of float64 rows."""
    x = np.asarray(x, np.float64)
    rows, V = x.shape
    lp, ent, ids, val = np.zeros(rows), np.zeros(rows), np.zeros((rows, top), np.int32), np.zeros((rows, top))
    for r in range(rows):
        y = x[r]
        order = np.argsort(np.where(np.isnan(y), -np.inf, -y), kind="stable")[:top]
        ids[r] = order
        with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
            if np.isnan(y).any() or (y == np.inf).any():
                lp[r] = ent[r] = np.nan
                val[r] = np.nan
                continue
            if (y == -np.inf).all():
                lp[r], ent[r], val[r] = -np.inf, 0, -np.inf
                lp[r] = -np.inf if 0 <= tokens[r] < V else np.nan
                continue
            m = y.max()
            e = np.exp(y - m)
            lse = m + np.log(e.sum())
            ent[r] = np.log(e.sum()) - np.where(e > 0, e * np.where(e > 0, y - m, 0), 0).sum() / e.sum()
            lp[r] = y[tokens[r]] - lse if 0 <= tokens[r] < V else np.nan
            val[r] = y[order] - lse
    return lp, ent, ids, val
