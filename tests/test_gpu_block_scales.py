"""Attention over the block-scaled cache (t2r_amd.ops) where the V blocks' scales lie far apart, against float64: a row's
result depends on the blocks that it sees and on nothing else, whatever their sizes."""
import math

import numpy as np
import pytest

from test_gpu_block import HALF, Both, F, env, i32, put, rounded  # noqa: F401 (env is the fixture)

pytestmark = pytest.mark.gpu
MAXF = float(np.finfo(F).max)


def rows_of(c, q, b, n_new, H, scale, only, w_half):
    """{row: (outputs [H * hd], bound)} in float64 of the rows `only` of sequence b, whose n_new newest are rows 0 .. n_new - 1 of
    q. With A the largest sum |q_i k_i| scale of a row, n the keys that it sees, p its probabilities:
      - scores in fp32 from q in two fp16 pieces: A (2^-22 + (hd + 8) 2^-24), twice (numerator and denominator), the exponent's
        argument A 2^-22 and exp2 2^-21, V's scale as a power of two 2^-22, the weights' two pieces 2^-21 and the sums
        (n / 8 + 128) 2^-24, all relative to sum p |v|;
      - a weight p vs is held with 2^11 put before the largest that the row sees, so fp16's last half step, 2^-25, is 2^-36 of that:
        n 2^-36 127 max(p vs) over the keys that it sees;
      - fp32's smallest half step.
    w_half: half a step of a weight that is one fp16 number (2^-11), of each key."""
    hd, Hk = c.host.hd, c.host.Hk
    n_all = int(c.lens[b])
    k, v, there = c.host.values(c.table, b, n_all)
    bs = c.host.bs
    blk = [int(c.table[b][j]) for j in range(-(-n_all // bs))]
    vs = np.repeat(np.stack([c.host.vs[x].astype(np.float64) if x >= 0 else np.zeros(Hk) for x in blk]), bs, axis=0)[:n_all]
    out = {}
    for r in only:
        n = n_all - n_new + r + 1
        ok = there[:n]
        y, tol = np.zeros(H * hd), np.zeros(H * hd)
        for h in range(H):
            g = h * Hk // H
            kk, vv, ss = k[:n, g][ok], v[:n, g][ok], vs[:n, g][ok]
            x = np.asarray(q[r], np.float64).reshape(H, hd)[h]
            s = kk @ x * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            A = (np.abs(kk) @ np.abs(x)).max() * scale
            rel = 2 * A * (2.0 ** -22 + (hd + 8) * 2.0 ** -24) + A * 2.0 ** -22 + 2.0 ** -20 + 2.0 ** -21 + (n / 8 + 128) * 2.0 ** -24 + w_half
            at = slice(h * hd, (h + 1) * hd)
            y[at] = p @ vv
            tol[at] = rel * (p @ np.abs(vv)) + n * 2.0 ** -36 * 127 * (p * ss).max() + 2.0 ** -149
        out[r] = (y, tol)
    return out


def compare(got, want, dtype):
    g = got.double().cpu().numpy()
    for r, (y, tol) in want.items():
        t = tol + HALF[dtype] * np.abs(y) * 1.01 + (2.0 ** -25 if dtype == "f16" else 0)    # (fp16's smallest half step)
        off = np.abs(g[r] - y)
        i = int(np.argmax(np.where(np.isnan(off), np.inf, off - t)))
        assert (off <= t).all(), (r, i, g[r][i], y[i], off[i], t[i])


# H, Hk, hd, block, rows of the call, of which kernel
FORMS = [
    (8, 2, 64, 16, 8, "32 columns"),
    (4, 2, 128, 16, 70, "64 columns, hd 128"),
    (6, 2, 48, 32, 90, "64 columns"),
    (64, 16, 64, 16, 1100, "128 columns"),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("grow", [20, 40, 126])
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_rows_are_free_of_later_scales(env, form, grow, dtype):
    """The last block's V scale is 2^grow larger than the others': the rows before that block are what they are without it, by
    the ragged form and by the step form at their own lengths."""
    torch, ops = env
    H, Hk, hd, block, rows, _ = FORMS[form]
    rng = np.random.default_rng(form + grow)
    n = (rows + 2 * block) // block * block - block + 3                    # three tokens in the last block
    c = Both(torch, ops, rng, [n], Hk, hd, block).fill(rng)
    last = c.table[0, (n - 1) // block]
    c.host.vs[last] = np.minimum(c.host.vs[last].astype(np.float64) * 2.0 ** grow, MAXF / 127).astype(F)
    c.send()
    x, t = rounded(torch, rng.standard_normal((rows, H * hd)) * 1.5, dtype)
    got = ops.attention_block_prefill(t, *c.dev, i32(torch, [0, rows]), c.lens_d, H)
    free = rows - 3                                                        # rows that do not see the last block
    only = sorted({0, free // 2, max(free - 17, 0), free - 2, free - 1})
    want = rows_of(c, x, 0, rows, H, 1 / math.sqrt(hd), only, 0 if dtype == "f32" else 2.0 ** -11)
    compare(got, want, dtype)
    for r in only:
        step = ops.attention_block(t[r:r + 1], *c.dev, i32(torch, [n - rows + r + 1]), H)
        compare(step, {0: want[r]}, dtype)


def test_rows_before_an_infinity(env):
    """An infinity among V's rows is stored as the largest float: the rows of earlier blocks keep their results, those that see
    it give finite ones."""
    torch, ops = env
    rng = np.random.default_rng(31)
    H, Hk, hd, block, n = 4, 2, 64, 16, 67
    c = Both(torch, ops, rng, [n], Hk, hd, block).send()
    x = rng.standard_normal((n, (H + 2 * Hk) * hd)).astype(F)
    x[65, -5] = np.inf
    t = put(torch, x)
    k, v, q = x[:, H * hd:(H + Hk) * hd], x[:, (H + Hk) * hd:], x[:, :H * hd]
    c.host.append(k, v, c.table, [0, n], c.lens)
    ops.kv_append_block(t[:, H * hd:(H + Hk) * hd], t[:, (H + Hk) * hd:], *c.dev, i32(torch, [0, n]), c.lens_d)
    c.same()
    got = ops.attention_block_prefill(t[:, :H * hd], *c.dev, i32(torch, [0, n]), c.lens_d, H)
    compare(got, rows_of(c, q, 0, n, H, 1 / math.sqrt(hd), (0, 15, 16, 40, 63, 64, 65, 66), 0), "f32")
    step = ops.attention_block(t[n - 1:, :H * hd], *c.dev, c.lens_d, H)
    compare(step, {0: rows_of(c, q[n - 1:], 0, 1, H, 1 / math.sqrt(hd), (0,), 0)[0]}, "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("form", ["step", "step in parts", "few", "few in parts", "tile", "tile over segments"])
def test_weights_against_scales(env, form, dtype):
    """Scores that spread over e^50 and V scales that spread over 2^240, among them zero and subnormal ones: what a row adds up is
    held against the largest product of a probability and a scale, not against the largest scale; and each row's own block
    carries next to all of its weight however small its values are."""
    torch, ops = env
    H, Hk, hd, block = 8, 2, 64, 16
    n, width, rows = {"step": (333, None, 1), "step in parts": (3000, 512, 1), "few": (333, None, 7), "few in parts": (3000, 256, 7),
                      "tile": (333, None, 100), "tile over segments": (4300, None, 90)}[form]
    rng = np.random.default_rng(len(form))
    c = Both(torch, ops, rng, [n], Hk, hd, block, width=width).fill(rng)
    c.host.vs[:] = np.exp2(rng.uniform(-140, 100, c.host.vs.shape))
    z = c.table[0, 3]
    c.host.vc[z] = 0
    c.host.vs[z] = 0
    c.send()
    x, t = rounded(torch, rng.standard_normal((rows, H * hd)) * rng.choice([0.3, 3, 12], (rows, 1)), dtype)
    if form.startswith("step"):
        got = ops.attention_block(t, *c.dev, c.lens_d, H)
    else:
        got = ops.attention_block_prefill(t, *c.dev, i32(torch, [0, rows]), c.lens_d, H)
    only = sorted({0, rows // 3, rows // 2, rows - 1})
    compare(got, rows_of(c, x, 0, rows, H, 1 / math.sqrt(hd), only, 0 if dtype == "f32" else 2.0 ** -11), dtype)


@pytest.mark.parametrize("size", [1e36, 3e37, 1e-37, 1e-41])
@pytest.mark.parametrize("form", ["step", "step in parts", "few", "few in parts", "tile", "tile in parts"])
def test_values_at_the_ends_of_the_range(env, form, size):
    """V near fp32's largest and smallest numbers, of all keys: their weighted mean is in range and so is every result."""
    torch, ops = env
    H, Hk, hd, block = 8, 2, 64, 64
    n, width, rows = {"step": (50, None, 1), "step in parts": (5000, None, 1), "few": (50, None, 5), "few in parts": (5000, None, 5),
                      "tile": (200, None, 100), "tile in parts": (2500, None, 300)}[form]
    rng = np.random.default_rng(41)
    c = Both(torch, ops, rng, [n], Hk, hd, block, width=width).fill(rng)
    c.host.vs[:] = (rng.uniform(0.5, 1, c.host.vs.shape) * size / 127).astype(F)
    c.send()
    x = rng.standard_normal((rows, H * hd)).astype(F)
    t = put(torch, x)
    if form.startswith("step"):
        got = ops.attention_block(t, *c.dev, c.lens_d, H)
    else:
        got = ops.attention_block_prefill(t, *c.dev, i32(torch, [0, rows]), c.lens_d, H)
    assert torch.isfinite(got).all()
    only = sorted({0, rows // 2, rows - 1})
    compare(got, rows_of(c, x, 0, rows, H, 1 / math.sqrt(hd), only, 0), "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("form", ["step", "few", "tile"])
def test_scores_up_to_millions(env, form, dtype):
    """Scores up to 1.9 million, rising along the keys so that the bases are raised again and again, one key far above the rest:
    its value is the result (the others' weights are below e^-1000)."""
    torch, ops = env
    H, Hk, hd, block, n = 4, 2, 64, 64, 300
    rows = {"step": 1, "few": 4, "tile": 80}[form]
    rng = np.random.default_rng(51)
    c = Both(torch, ops, rng, [n], Hk, hd, block).fill(rng, spread=2.0)
    c.host.ks[:] = 1
    sign = rng.choice([-1, 1], hd)
    top = n - rows                                                         # (every row sees it)
    for j in range(n):
        c.host.kc[c.table[0, j // block], :, j % block] = sign * (j * 100 // n if j != top else 127)
    c.send()
    x, t = rounded(torch, np.tile(sign * 1.9e6 * 8 / (127 * hd), (rows, H)), dtype)
    if form == "step":
        got = ops.attention_block(t, *c.dev, c.lens_d, H)
    else:
        got = ops.attention_block_prefill(t, *c.dev, i32(torch, [0, rows]), c.lens_d, H)
    _, v, _ = c.host.values(c.table, 0, n)
    y = np.repeat(v[top], H // Hk, axis=0).reshape(-1)
    # A weight alone in l and o: its pieces and the sums at most 2^-11. Its exponent's addend is u - M, with u the V scale's log2 and
    # M a whole number of the scores' size: log2(e) 1.9e6 < 2^22, where half a step of fp32 is 2^-3, and u's fraction is rounded
    # to that once, in o and not in l: up to 2^(2^-3) - 1 = 0.0906 of the result (the term A 2^-22 of rows_of at this A is 0.45).
    tol = np.abs(y) * (0.0906 + 2.0 ** -10)
    compare(got, {r: (y, tol) for r in (0, rows - 1)}, dtype)


@pytest.mark.parametrize("form,dtype", [("step", "f16"), ("step", "bf16"), ("step of wide groups", "f16"), ("step of wide groups", "bf16"),
                                        ("few", "f16"), ("few, hd 128", "f16"), ("tile", "f16"), ("tile, hd 128", "f16"),
                                        ("wide tile", "f16")])
def test_weights_keep_their_bits_in_16_bit_rows(env, form, dtype):
    """Rows of 16 bits whose weights are held in two fp16 pieces, as fp32 rows' are: the result is the exact one rounded once, up
    to fp32's own errors. (q in one piece loses 2^-25 of a row's largest value where a value is small: below A 2^-22 in a score.)"""
    torch, ops = env
    H, Hk, hd, n, rows = {"step": (32, 8, 64, 400, 1), "step of wide groups": (32, 2, 128, 300, 1), "few": (8, 2, 64, 300, 8),
                          "few, hd 128": (8, 2, 128, 300, 8), "tile": (8, 2, 64, 200, 150), "tile, hd 128": (8, 4, 128, 200, 150),
                          "wide tile": (32, 8, 64, 2200, 2100)}[form]
    rng = np.random.default_rng(61)
    c = Both(torch, ops, rng, [n], Hk, hd, 64).fill(rng).send()
    x, t = rounded(torch, rng.standard_normal((rows, H * hd)), dtype)
    if form.startswith("step"):
        got = ops.attention_block(t, *c.dev, c.lens_d, H)
    else:
        got = ops.attention_block_prefill(t, *c.dev, i32(torch, [0, rows]), c.lens_d, H)
    only = range(rows) if rows <= 8 else (0, 1, 33, rows // 2, rows - 2, rows - 1)
    for r, (y, tol) in rows_of(c, x, 0, rows, H, 1 / math.sqrt(hd), only, 0).items():
        # (between the roundings of the exact value less and more what fp32 is off; 2^-24 of it: the result's own rounding to fp32)
        tol = tol + np.abs(y) * 2.0 ** -24
        lo, hi = (rounded(torch, v, dtype)[0] for v in (y - tol, y + tol))
        g = got[r].double().cpu().numpy()
        bad = (g < lo) | (g > hi)
        assert not bad.any(), (r, int(bad.sum()), g[bad][:3], y[bad][:3], tol[bad][:3])
