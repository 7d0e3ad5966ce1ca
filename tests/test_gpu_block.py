"""The block-scaled KV cache, the attention over it and the log probabilities (t2r_amd.ops) against float64 (blockref)."""
import math

import numpy as np
import pytest

from blockref import Cache, attention, logprobs

pytestmark = pytest.mark.gpu

F = np.float32
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}           # half a step, relative


@pytest.fixture(scope="module")
def env():
    import torch

    from t2r_amd import abi, ops
    abi.load()
    return torch, ops


def dt(torch, name):
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def put(torch, a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).to("cuda:0")
    return t if dtype is None else t.to(dtype)


def i32(torch, a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda:0")


def rounded(torch, x, dtype):
    """x as the type holds it (float64), and the tensor."""
    t = put(torch, x.astype(F), dt(torch, dtype))
    return t.double().cpu().numpy(), t


class Both:
    """The same cache on the host and on the device, with a shuffled table."""

    def __init__(self, torch, ops, rng, lens, Hk, hd, block, width=None, spare=2):
        self.torch, self.ops = torch, ops
        used = [-(-max(int(n), 0) // block) for n in lens]
        width = width or max(max(used), 1)
        n = sum(min(u, width) for u in used) + spare
        order = rng.permutation(n)
        self.table = np.full((len(lens), width), -1, np.int32)
        at = 0
        for b, u in enumerate(used):
            u = min(u, width)
            self.table[b, :u] = order[at:at + u]
            at += u
        self.host = Cache(n, Hk, hd, block)
        self.lens = np.asarray(lens, np.int32)

    def fill(self, rng, spread=1.0):
        h = self.host
        h.kc[:] = np.clip(np.rint(rng.standard_normal(h.kc.shape) * 35), -127, 127)
        h.vc[:] = np.clip(np.rint(rng.standard_normal(h.vc.shape) * 35), -127, 127)
        h.ks[:] = np.exp(rng.standard_normal(h.ks.shape) * 0.4 * spread) / 35
        h.vs[:] = np.exp(rng.standard_normal(h.vs.shape) * spread) / 35
        return self

    def send(self):
        h = self.host
        self.dev = [put(self.torch, a) for a in (h.kc, h.vc, h.ks, h.vs, self.table)]
        self.lens_d = i32(self.torch, self.lens)
        return self

    def same(self):
        h = self.host
        for name, want, got in zip(("ks", "vs", "kc", "vc"), (h.ks, h.vs, h.kc, h.vc), (self.dev[2], self.dev[3], self.dev[0], self.dev[1])):
            g = got.cpu().numpy()
            assert np.array_equal(g, want), (name, int((g != want).sum()), np.argwhere(g != want)[:5].tolist())


# ------------------------------------------------------------------ rows into the cache
APPENDS = [
    # block, Hk, hd, news, lens
    (64, 8, 64, [1] * 5, [1, 64, 65, 100, 129]),
    (16, 3, 48, [7, 0, 33, 1], [7, 20, 50, 17]),
    (32, 2, 16, [40], [40]),
    (128, 1, 128, [300, 129], [300, 257]),
    (16, 6, 48, [16, 17, 15], [32, 33, 31]),
    (64, 5, 96, [2, 3], [66, 64]),
    (64, 1, 80, [1], [1]),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append_codes_and_scales(env, case, dtype):
    """Codes and scales are those of the definition, bit for bit; the rows are columns of a wider matrix; a second call
    continues the sequences, with larger values (scales grow), then smaller ones (they stay)."""
    torch, ops = env
    block, Hk, hd, news, lens = APPENDS[case]
    rng = np.random.default_rng(case)
    n = Hk * hd
    last = np.asarray(lens) + np.asarray(news) * 2
    c = Both(torch, ops, rng, last, Hk, hd, block).fill(rng).send()
    starts = np.concatenate([[0], np.cumsum(news)])
    for step, amp in enumerate((1.0, 3.0, 0.2)):
        ln = np.asarray(lens) + np.asarray(news) * step
        x, t = rounded(torch, rng.standard_normal((starts[-1], 3 + 2 * n + 1)) * amp, dtype)
        c.host.append(x[:, 3:3 + n], x[:, 3 + n:3 + 2 * n], c.table, starts, ln)
        ops.kv_append_block(t[:, 3:3 + n], t[:, 3 + n:3 + 2 * n], *c.dev, i32(torch, starts), i32(torch, ln))
        c.same()


def test_append_borders(env):
    """Values at and next to the half steps of a scale that is no power of two, zeros, the largest and smallest floats,
    infinities and NaN."""
    torch, ops = env
    rng = np.random.default_rng(5)
    Hk, hd, block = 2, 64, 64
    rows = 64
    x = np.zeros((rows, 2, Hk, hd), F)
    m = F(3.7)
    s = F(m / F(127))
    half = (rng.integers(-127, 127, (rows, Hk, hd)) + 0.5) * float(s)
    x[:, 0] = np.nextafter(half.astype(F), rng.choice([-np.inf, np.inf], half.shape).astype(F))
    x[:, 0, :, :9] = half.astype(F)[:, :, :9]
    x[0, 0, :, 0] = m
    x[:, 1] = rng.standard_normal((rows, Hk, hd)) * np.exp(rng.uniform(-90, 80, (rows, Hk, hd)))
    x[5, 1, 0, 3], x[6, 1, 0, 4], x[7, 1, 1, 5] = np.inf, -np.inf, np.nan
    for case in range(3):
        if case == 1:
            x *= F(1e-38)                                                  # subnormal values and scales
            x[:, 1] = rng.standard_normal((rows, Hk, hd)) * 1e-44
        if case == 2:
            x[:] = 0
            x[3, 0] = np.nan
        c = Both(torch, ops, rng, [rows], Hk, hd, block).send()
        t = put(torch, x.reshape(rows, -1))
        c.host.append(x[:, 0], x[:, 1], c.table, [0, rows], c.lens)
        ops.kv_append_block(t[:, :Hk * hd], t[:, Hk * hd:], *c.dev, i32(torch, [0, rows]), c.lens_d)
        c.same()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("top", [127.0, 1.875, 1.9765625, 0.0234375, 127 * 2.0 ** -12])
def test_append_halves_of_16_bit_rows(env, dtype, top):
    """Ties (scales that are powers of two) and values a rounding beside them (half of the largest value, 63.5 steps but for the
    scale's rounding), with zeros, infinities and NaN among them, into empty and partly filled blocks."""
    torch, ops = env
    rng = np.random.default_rng(23)
    Hk, hd, block, rows = 2, 64, 32, 50
    x = rng.choice(np.r_[np.arange(-63, 63) + 0.5, -63.5, 63.5, 127, -127, 0, 21.5, 42.25, 31.75], (rows, 2, Hk, hd)) * (top / 127)
    x[0] = top
    x, t = rounded(torch, x.reshape(rows, -1), dtype)
    c = Both(torch, ops, rng, [rows + 7], Hk, hd, block).send()
    n = Hk * hd
    for r0, r1, at in ((0, 7, 7), (0, rows, rows + 7)):
        if r1 == rows:
            t[9, 3], t[11, n + 5], t[12, 8] = np.inf, -np.inf, np.nan
            x = t.double().cpu().numpy()
        c.host.append(x[r0:r1, :n].astype(F), x[r0:r1, n:].astype(F), c.table, [0, r1 - r0], [at])
        ops.kv_append_block(t[r0:r1, :n], t[r0:r1, n:], *c.dev, i32(torch, [0, r1 - r0]), i32(torch, [at]))
        c.same()


def test_append_places_without_a_block(env):
    """Rows below position 0, past the table, and at table entries outside the pool are dropped; slots behind the rows and
    other blocks keep what they hold; rows of no sequence are left out."""
    torch, ops = env
    rng = np.random.default_rng(6)
    Hk, hd, block = 2, 32, 16
    c = Both(torch, ops, rng, [40, 40, 40], Hk, hd, block).fill(rng)
    c.table[1, 1] = c.host.n                                                # one past the pool
    c.table[2, 0] = -7
    c.send()
    starts, lens = [0, 45, 85, 95], [40, 40, 52]                           # 5 rows below 0; 4 rows past the table of 48
    x = rng.standard_normal((99, 2, Hk * hd)).astype(F)
    t = put(torch, x)
    c.host.append(x[:, 0], x[:, 1], c.table, starts, lens)
    ops.kv_append_block(t[:, 0], t[:, 1], *c.dev, i32(torch, starts), i32(torch, lens))
    c.same()
    k, v = ops.kv_read_block(*c.dev, i32(torch, starts), i32(torch, lens), 95)
    want_k, want_v = np.zeros((95, Hk * hd)), np.zeros((95, Hk * hd))
    for r, blk, slot, p, b in c.host.places(c.table, starts, lens, 95):
        if blk >= 0:
            want_k[r] = (c.host.kc[blk, :, slot].astype(F) * c.host.ks[blk][:, None]).reshape(-1)
            want_v[r] = (c.host.vc[blk, :, :, slot].astype(F) * c.host.vs[blk][:, None]).reshape(-1)
    assert np.array_equal(k.cpu().numpy(), want_k.astype(F)) and np.array_equal(v.cpu().numpy(), want_v.astype(F))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("block,Hk,hd", [(16, 3, 48), (64, 8, 64), (128, 2, 128), (32, 1, 16)])
def test_read_gives_the_values(env, block, Hk, hd, dtype):
    torch, ops = env
    rng = np.random.default_rng(block)
    lens, news = [block * 2 + 5, 3, block, 0], [block * 2 + 5, 1, block - 1, 0]
    c = Both(torch, ops, rng, lens, Hk, hd, block).fill(rng).send()
    starts = np.concatenate([[0], np.cumsum(news)])
    k, v = ops.kv_read_block(*c.dev, i32(torch, starts), c.lens_d, int(starts[-1]), dtype=dt(torch, dtype))
    for b, n in enumerate(lens):
        kk, vv, _ = c.host.values(c.table, b, n)
        for got, want in ((k, kk), (v, vv)):
            w = put(torch, want[n - news[b]:].reshape(news[b], Hk * hd).astype(F), dt(torch, dtype))
            assert torch.equal(got[starts[b]:starts[b + 1]], w)


# ------------------------------------------------------------------ attention
def check(torch, got, want, bound, dtype):
    g = got.double().cpu().numpy()
    there = ~np.isnan(want[:, 0])
    assert np.isfinite(g[there]).all()
    g, want, bound = g[there], want[there], bound[there]
    off = np.abs(g - want)
    tol = bound + HALF[dtype] * np.abs(want) * 1.01 + (2.0 ** -25 if dtype == "f16" else 0)    # (fp16's smallest half step)
    worst = np.unravel_index(np.argmax(off - tol), off.shape)
    assert (off <= tol).all(), (worst, g[worst], want[worst], off[worst], tol[worst])


STEPS = [
    # H, Hk, hd, block, lens, width
    (9, 3, 64, 64, [96], 32),
    (32, 8, 64, 64, [1, 63, 64, 65, 0, 300, 255, 256, 257], None),
    (16, 8, 128, 32, [700, 1], 64),
    (6, 6, 48, 16, [1, 2, 15, 16, 17, 31, 33, 255], 16),
    (12, 4, 80, 128, [130, 513], None),
    (8, 1, 96, 16, [49], None),
    (16, 1, 32, 64, [200, 100], None),
    (32, 1, 128, 64, [321], None),
    (4, 2, 16, 16, [2100], None),
    (7, 7, 112, 64, [70, 400], None),
    (24, 2, 64, 32, [1100, 40], 128),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", range(len(STEPS)))
def test_attention_step(env, case, dtype):
    torch, ops = env
    H, Hk, hd, block, lens, width = STEPS[case]
    rng = np.random.default_rng(100 + case)
    c = Both(torch, ops, rng, lens, Hk, hd, block, width=width).fill(rng).send()
    x, t = rounded(torch, rng.standard_normal((len(lens), H * hd + 5)) * 1.5, dtype)
    got = ops.attention_block(t[:, 5:], *c.dev, c.lens_d, H)
    starts = list(range(len(lens) + 1))
    want, bound = attention(c.host, x[:, 5:], c.table, starts, lens, H, 1 / math.sqrt(hd), 0 if dtype == "f32" else 2.0 ** -11)
    check(torch, got, want, bound, dtype)
    assert not got[np.asarray(lens) == 0].any()


ROWS = [
    # H, Hk, hd, block, news, lens, width
    (16, 8, 128, 64, [130], [130], None),
    (9, 3, 64, 16, [33, 1, 0, 70], [33, 90, 10, 200], None),
    (32, 8, 64, 64, [8, 8], [900, 333], 64),
    (6, 6, 48, 32, [65], [100], None),
    (12, 4, 80, 128, [5, 64], [5, 64], None),
    (8, 1, 96, 16, [20], [20], 300),
    (32, 1, 64, 64, [3, 40], [70, 41], None),
    (4, 2, 16, 16, [100], [2500], None),
    (7, 7, 112, 64, [31], [31], None),
    (20, 2, 128, 32, [17], [300], None),
    (8, 2, 64, 64, [50, 0, 1, 0, 0, 2, 0, 0], [700, 5, 1, 0, 9, 2000, 3, 3], 64),      # (few rows in all, but not of the first)
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", range(len(ROWS)))
def test_attention_rows(env, case, dtype):
    torch, ops = env
    H, Hk, hd, block, news, lens, width = ROWS[case]
    rng = np.random.default_rng(200 + case)
    c = Both(torch, ops, rng, lens, Hk, hd, block, width=width).fill(rng).send()
    starts = np.concatenate([[0], np.cumsum(news)])
    x, t = rounded(torch, rng.standard_normal((starts[-1], H * hd + 3)) * 1.5, dtype)
    got = ops.attention_block_prefill(t[:, 3:], *c.dev, i32(torch, starts), c.lens_d, H)
    want, bound = attention(c.host, x[:, 3:], c.table, starts, lens, H, 1 / math.sqrt(hd), 0 if dtype == "f32" else 2.0 ** -11)
    check(torch, got, want, bound, dtype)


@pytest.mark.parametrize("form", ["step", "rows"])
def test_attention_far_apart_scales(env, form):
    """Blocks whose scales differ by many orders (a zero block among them), rows of very large and very small q, and scores
    that leave one key only."""
    torch, ops = env
    rng = np.random.default_rng(7)
    H, Hk, hd, block = 4, 2, 64, 16
    n = 333
    c = Both(torch, ops, rng, [n], Hk, hd, block).fill(rng)
    c.host.vs[:] = np.exp(rng.uniform(-60, 10, c.host.vs.shape))
    c.host.ks[:] = np.exp(rng.uniform(-6, 1, c.host.ks.shape)) / 35
    z = c.table[0, 3]
    c.host.kc[z] = c.host.vc[z] = 0
    c.host.ks[z] = c.host.vs[z] = 0
    c.send()
    rows = 1 if form == "step" else 9
    x = rng.standard_normal((rows, H, hd)).astype(F)
    x[:, 0] *= F(1e-30)
    x[:, 1] *= F(40)
    x[:, 2] = 0
    t = put(torch, x.reshape(rows, -1))
    if form == "step":
        got = ops.attention_block(t, *c.dev, c.lens_d, H)
    else:
        got = ops.attention_block_prefill(t, *c.dev, i32(torch, [0, rows]), c.lens_d, H)
    want, bound = attention(c.host, x, c.table, [0, rows], [n], H, 1 / math.sqrt(hd))
    check(torch, got, want, bound, "f32")


@pytest.mark.parametrize("form", ["step", "rows"])
def test_attention_holes_and_ends(env, form):
    """Table entries outside the pool leave their positions out; positions past the table do not count; a sequence all of
    holes gives zeros, rows below position 0 give NaN; stale codes behind a sequence's end do nothing."""
    torch, ops = env
    rng = np.random.default_rng(8)
    H, Hk, hd, block = 6, 2, 48, 16
    lens = [50, 100, 32, 7]
    c = Both(torch, ops, rng, lens, Hk, hd, block, width=5).fill(rng)
    c.table[0, 1] = c.host.n + 3
    c.table[2, :] = -1
    tail = c.table[0, 3]                                                     # 50 = 3 * 16 + 2: 14 stale slots
    c.host.kc[tail, :, 2:] = 127
    c.host.vc[tail, :, :, 2:] = -127
    c.send()
    news = [1] * 4 if form == "step" else [5, 30, 3, 9]
    starts = np.concatenate([[0], np.cumsum(news)])
    x = rng.standard_normal((starts[-1], H * hd)).astype(F)
    t = put(torch, x)
    if form == "step":
        got = ops.attention_block(t, *c.dev, c.lens_d, H)
    else:
        got = ops.attention_block_prefill(t, *c.dev, i32(torch, starts), c.lens_d, H)
    want, bound = attention(c.host, x, c.table, starts, lens, H, 1 / math.sqrt(hd))
    check(torch, got, want, bound, "f32")
    assert not got[starts[2]:starts[3]].any()
    if form == "rows":
        assert torch.isnan(got[starts[3]:starts[3] + 2]).all() and torch.isfinite(got[:starts[3]]).all()


def test_attention_nan_stays_in_its_row(env):
    torch, ops = env
    rng = np.random.default_rng(9)
    H, Hk, hd = 8, 2, 64
    c = Both(torch, ops, rng, [70, 200], Hk, hd, 64).fill(rng).send()
    x = rng.standard_normal((2, H, hd)).astype(F)
    x[1, 3, 5] = np.nan
    got = ops.attention_block(put(torch, x.reshape(2, -1)), *c.dev, c.lens_d, H).view(2, H, hd).cpu().numpy()
    bad = np.isnan(got).any(-1)
    assert bad[1, 3] and bad.sum() == 1
    y = rng.standard_normal((40, H, hd)).astype(F)
    y[11, 6, 0] = np.nan
    got = ops.attention_block_prefill(put(torch, y.reshape(40, -1)), *c.dev, i32(torch, [0, 20, 40]), c.lens_d, H)
    bad = np.isnan(got.view(40, H, hd).cpu().numpy()).any(-1)
    assert bad[11, 6] and bad.sum() == 1


def test_step_and_rows_agree_on_long_caches(env):
    """A cache past the segment of 2048 keys that the ragged form keeps its tables of, one row, both forms."""
    torch, ops = env
    rng = np.random.default_rng(10)
    H, Hk, hd = 8, 4, 128
    n = 5000
    c = Both(torch, ops, rng, [n], Hk, hd, 64).fill(rng, spread=2.0).send()
    x = rng.standard_normal((1, H * hd)).astype(F)
    want, bound = attention(c.host, x, c.table, [0, 1], [n], H, 0.05)
    check(torch, ops.attention_block(put(torch, x), *c.dev, c.lens_d, H, scale=0.05), want, bound, "f32")
    check(torch, ops.attention_block_prefill(put(torch, x), *c.dev, i32(torch, [0, 1]), c.lens_d, H, scale=0.05), want, bound, "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("Hk,hd", [(32, 64), (32, 128), (48, 16)])
def test_rows_over_several_segments(env, Hk, hd, dtype):
    """Enough tiles that none is cut along its keys, over caches of several segments whose largest scales differ: every
    tile passes from segment to segment. A few rows are compared."""
    torch, ops = env
    rng = np.random.default_rng(17)
    lens, news = [4500, 2100], [700, 400]
    H = Hk
    c = Both(torch, ops, rng, lens, Hk, hd, 64).fill(rng)
    for b in range(2):
        c.host.vs[c.table[b, :32]] *= F(0.01)                              # the later segments' scales are larger
    c.send()
    starts = np.concatenate([[0], np.cumsum(news)])
    x, t = rounded(torch, rng.standard_normal((starts[-1], H * hd)), dtype)
    got = ops.attention_block_prefill(t, *c.dev, i32(torch, starts), c.lens_d, H)
    want, bound = attention(c.host, x, c.table, starts, lens, H, 1 / math.sqrt(hd), 0 if dtype == "f32" else 2.0 ** -11,
                            only=(0, 63, 333, 699, 700, 1047, 1048, 1099))
    check(torch, got, want, bound, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("H,Hk,hd,block,news,lens", [
    (32, 8, 64, 64, [2100], [2100]),
    (30, 3, 48, 32, [1203, 1, 0, 1500], [1300, 70, 10, 3000]),               # (10 heads a group: 12 rows a tile of 128 columns)
    (96, 3, 16, 16, [33, 700], [33, 2500]),
])
def test_many_rows(env, H, Hk, hd, block, news, lens, dtype):
    """Prompts long enough for the widest tiles at small head dims. A few rows are compared, each tile's end among them."""
    torch, ops = env
    rng = np.random.default_rng(18)
    c = Both(torch, ops, rng, lens, Hk, hd, block).fill(rng, spread=1.5).send()
    starts = np.concatenate([[0], np.cumsum(news)])
    rows = int(starts[-1])
    assert rows * H > 64 * 1024
    x, t = rounded(torch, rng.standard_normal((rows, H * hd)), dtype)
    got = ops.attention_block_prefill(t, *c.dev, i32(torch, starts), c.lens_d, H)
    rt = 128 * Hk // H
    only = sorted({r for r in (0, rt - 1, rt, 2 * rt - 1, 32, 700, news[0] - 1, news[0], rows // 2, rows - rt - 1, rows - 2, rows - 1)})
    want, bound = attention(c.host, x, c.table, starts, lens, H, 1 / math.sqrt(hd), 0 if dtype == "f32" else 2.0 ** -11, only=only)
    check(torch, got, want, bound, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("H,Hk,hd,block,news,lens,width", [
    (32, 8, 64, 64, [548], [4500], 128),
    (16, 8, 128, 32, [300, 0, 251], [3300, 40, 2900], 256),
    (32, 8, 48, 128, [270, 33], [3000, 33], 32),                             # (one of them within the first part)
])
def test_turns_late_in_long_caches(env, H, Hk, hd, block, news, lens, width, dtype):
    """Some hundred rows, whose tiles' keys are cut into a few long parts. A few rows are compared."""
    torch, ops = env
    rng = np.random.default_rng(24)
    c = Both(torch, ops, rng, lens, Hk, hd, block, width=width).fill(rng, spread=1.5).send()
    starts = np.concatenate([[0], np.cumsum(news)])
    rows = int(starts[-1])
    x, t = rounded(torch, rng.standard_normal((rows, H * hd)), dtype)
    got = ops.attention_block_prefill(t, *c.dev, i32(torch, starts), c.lens_d, H)
    only = sorted({0, 15, 16, news[0] - 1, min(news[0], rows - 1), rows - 2, rows - 1})
    want, bound = attention(c.host, x, c.table, starts, lens, H, 1 / math.sqrt(hd), 0 if dtype == "f32" else 2.0 ** -11, only=only)
    check(torch, got, want, bound, dtype)


def test_many_sequences_with_few_rows(env):
    """More sequences than a wave has lanes, most of them without rows."""
    torch, ops = env
    rng = np.random.default_rng(11)
    H, Hk, hd, B = 4, 2, 32, 150
    lens = rng.integers(0, 40, B)
    news = np.where(rng.random(B) < 0.4, np.minimum(rng.integers(1, 9, B), lens), 0)
    c = Both(torch, ops, rng, lens, Hk, hd, 16).fill(rng).send()
    starts = np.concatenate([[0], np.cumsum(news)])
    rows = int(starts[-1])
    kv = rng.standard_normal((rows, 2, Hk * hd)).astype(F)
    t = put(torch, kv)
    c.host.append(kv[:, 0], kv[:, 1], c.table, starts, lens)
    ops.kv_append_block(t[:, 0], t[:, 1], *c.dev, i32(torch, starts), c.lens_d)
    c.same()
    x = rng.standard_normal((rows, H * hd)).astype(F)
    got = ops.attention_block_prefill(put(torch, x), *c.dev, i32(torch, starts), c.lens_d, H)
    want, bound = attention(c.host, x, c.table, starts, lens, H, 1 / math.sqrt(hd))
    check(torch, got, want, bound, "f32")


def test_offsets_past_32_bits(env):
    """A pool of over 2^31 bytes of codes, the sequence in its last blocks."""
    torch, ops = env
    rng = np.random.default_rng(12)
    H, Hk, hd, block, n = 16, 8, 128, 64, 200
    pool = (1 << 31) // (Hk * block * hd) + 40
    kc, vc, ks, vs = ops.block_cache(pool, Hk, hd, block)
    c = Cache(4, Hk, hd, block)
    table = np.arange(4)[None]
    x = rng.standard_normal((n, (H + 2 * Hk) * hd)).astype(F)
    c.append(x[:, H * hd:(H + Hk) * hd], x[:, (H + Hk) * hd:], table, [0, n], [n])
    t, far, st, ln = put(torch, x), i32(torch, table + pool - 4), i32(torch, [0, n]), i32(torch, [n])
    ops.kv_append_block(t[:, H * hd:(H + Hk) * hd], t[:, (H + Hk) * hd:], kc, vc, ks, vs, far, st, ln)
    for got, want in ((kc, c.kc), (vc, c.vc), (ks, c.ks), (vs, c.vs)):
        assert np.array_equal(got[-4:].cpu().numpy(), want)
        assert not got[:-4].view(torch.int8).any() if got.dtype == torch.int8 else not got[:-4].any()
    last = t[-1:, :H * hd]
    want, bound = attention(c, x[-1:, :H * hd], table, [0, 1], [n], H, 1 / math.sqrt(hd))
    check(torch, ops.attention_block(last, kc, vc, ks, vs, far, ln, H), want, bound, "f32")
    check(torch, ops.attention_block_prefill(last, kc, vc, ks, vs, far, i32(torch, [0, 1]), ln, H), want, bound, "f32")


# ------------------------------------------------------------------ log probabilities
def lp_check(torch, x, got, tokens, top, spans):
    """Sums of e^(x - m) over 32 values a thread and span, then a tree: (32 spans + 16) 2^-24 relative, the exponentials
    2^-22 each and |x - m| 2^-23 of their argument, weighted by them: D = sum p |x - m|, at most the entropy where m is the
    maximum and 4 more where it is a thread's (rows past a span: ln V > 9); m, ln l and x_t - lse are rounded."""
    lp, ent, ids, val = (None if t is None else t.cpu().numpy() for t in got)
    wl, we, wi, wv = logprobs(x, tokens, top)
    assert np.array_equal(ids, wi)
    y = np.where(np.isfinite(x), x, 0)
    big = np.abs(y).max(1)
    D = np.where(np.isfinite(we), we, 0) + 1 + np.log(x.shape[1])
    rel = (32 * spans + 16) * 2.0 ** -24 + 2.0 ** -22 + D * 2.0 ** -23
    tol = rel + 2.0 ** -22 * (big + D)
    for g, w, t in ((lp, wl, tol), (ent, we, 2 * D * rel + 2.0 ** -22 * D), (val, wv, tol[:, None])):
        fine = np.isfinite(w)
        assert np.array_equal(np.isnan(g), np.isnan(w)) and np.array_equal(g[~fine & ~np.isnan(w)], w[~fine & ~np.isnan(w)])
        t = np.broadcast_to(t, w.shape)
        assert (np.abs(g - w)[fine] <= t[fine] + 2.0 ** -23 * np.abs(w)[fine]).all(), float((np.abs(g - w)[fine] - t[fine]).max())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,V,top", [(1, 1, 1), (3, 61, 20), (2, 8192, 32), (5, 8193, 5), (4, 49155, 20), (2, 128256, 0), (33, 1000, 1),
                                        (1500, 40, 3), (700, 33000, 4)])
def test_logprobs(env, rows, V, top, dtype):
    torch, ops = env
    rng = np.random.default_rng(V + rows)
    x, t = rounded(torch, rng.standard_normal((rows, V + 3)) * 3, dtype)
    x, t = x[:, 3:], t[:, 3:]
    tokens = rng.integers(0, V, rows)
    tokens[0] = int(np.argmax(x[0]))
    lp_check(torch, x, ops.logprobs(t, i32(torch, tokens), top=top), tokens, top, 8)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [7, 8191, 8192, 8193, 8200, 16383, 16392])
def test_logprobs_starts_and_ends(env, V, dtype):
    """Rows at every alignment, around whole spans; the largest value first, last and at a span's ends."""
    torch, ops = env
    rng = np.random.default_rng(V)
    big, wide = rounded(torch, rng.standard_normal((9, V + 13)) * 2, dtype)
    for off in range(8):
        x, t = big[:, off:off + V].copy(), wide[:, off:off + V].clone()
        hot = [0, V - 1, min(8191, V - 1), min(8192, V - 1), min(8192 - off, V - 1), max(V - 8, 0), V // 2, 1, 6]
        x[np.arange(9), hot] = 11
        held = torch.empty_like(wide)
        held.fill_(float("nan"))                                       # (what lies beside the rows)
        held[:, off:off + V] = t
        held[torch.arange(9), off + torch.tensor(hot)] = 11
        got = ops.logprobs(held[:, off:off + V], i32(torch, hot), top=min(V, 6))
        lp_check(torch, x.astype(np.float64), got, np.asarray(hot), min(V, 6), 4)
        assert got[2][:, 0].tolist() == hot


def test_logprobs_odd_rows(env):
    """Banned values (-inf, the type's lowest), rows of nothing, of one value, of equal values, rising rows (every span beats
    the one before), NaN and +inf, tokens outside the vocabulary, -0 against +0."""
    torch, ops = env
    rng = np.random.default_rng(13)
    V = 20000
    x = (rng.standard_normal((11, V)) * 2).astype(F)
    x[0, rng.random(V) < 0.9] = -np.inf
    x[1] = -np.inf
    x[2] = -np.inf
    x[2, 12345] = 3
    x[3] = 1.5
    x[4] = np.arange(V) * 1e-3
    x[5, rng.random(V) < 0.5] = np.finfo(F).min
    x[6, 777] = np.nan
    x[7, 19999] = np.inf
    x[8] = np.where(rng.random(V) < 0.5, F(-0.0), F(0.0))
    x[9] = np.finfo(F).min
    tokens = np.asarray([int(np.flatnonzero(np.isfinite(x[0]))[0]), 5, 12345, 19999, 19999, 0, 1, 2, 3, 4, V])
    for top in (0, 1, 20, 32):
        lp_check(torch, x.astype(np.float64), ops.logprobs(put(torch, x), i32(torch, tokens), top=top), tokens, top, 3)
    assert ops.logprobs(put(torch, x))[0] is None


@pytest.mark.parametrize("rows", [13, 1030])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_logprobs_over_spans(env, rows, dtype):
    """A vocabulary of five whole spans of 8192 values and a rest, in a workgroup a span (few rows) or one for all: ranges
    banned with -inf or the type's lowest value, the largest values in the first, a middle, the last span, many of them or
    equal ones, rising and falling rows, a NaN and an infinity in later spans. The rows that differ are compared, and the last."""
    torch, ops = env
    rng = np.random.default_rng(19)
    V, S, low = 5 * 8192 + 40, 8192, float(torch.finfo(torch.bfloat16).min)
    x = (rng.standard_normal((13, V)) * 2).astype(F)
    x[0, :S] = -np.inf
    x[1, S:] = low
    x[2, :3 * S] = low
    x[3, 2 * S:3 * S] += 30
    x[4, 5 * S:] += 30
    x[5, :S] -= 40                                                     # all of the later spans beat the first
    x[6] = np.arange(V) * 2.0 ** -9
    x[7] = -np.arange(V) * 2.0 ** -9
    x[8, 300::100] = 9                                                 # (more equal ones than candidates are held, over the spans)
    x[9, 3 * S + 5] = np.nan
    x[10, 5 * S + 39] = np.inf
    x[11, S:2 * S] = -np.inf
    x[11, 4 * S:] = -np.inf
    x[11, 2 * S:4 * S] = low
    full = np.concatenate([x, (rng.standard_normal((rows - 13, V))).astype(F)])
    full, t = rounded(torch, full, dtype)
    tokens = rng.integers(0, V, rows)
    look = sorted({*range(13), rows - 1})
    for top in (0, 5, 32):
        got = ops.logprobs(t, i32(torch, tokens), top=top)
        lp_check(torch, full[look].astype(np.float64), tuple(g[look] for g in got), tokens[look], top, 6)


# ------------------------------------------------------------------ calls as programs make them
def serving_step(torch, ops, c, w, qkv, starts, lens, H, hd, Hk, step):
    """Append, attend, a linear layer to logits, and the answers' log probabilities."""
    q, n = H * hd, Hk * hd
    ops.kv_append_block(qkv[:, q:q + n], qkv[:, q + n:], *c, starts, lens)
    att = ops.attention_block(qkv[:, :q], *c, lens, H) if step else ops.attention_block_prefill(qkv[:, :q], *c, starts, lens, H)
    xq, s = ops.quant_act(att)
    logits = ops.linear(*w, xq, s)
    tok = ops.argmax(logits)
    return (att, logits, tok, *ops.logprobs(logits, tok, top=5))


def test_run_of_them_together(env):
    """Two prompts, then 40 tokens each: the cache, the attention over it and the answers stay those of the definitions."""
    torch, ops = env
    rng = np.random.default_rng(14)
    H, Hk, hd, V = 8, 2, 64, 500
    q, n = H * hd, Hk * hd
    c = Both(torch, ops, rng, [120, 120], Hk, hd, 32).send()
    w = (put(torch, rng.integers(-127, 128, (V, q)).astype(np.int8)), put(torch, (rng.random(V) * 0.01 + 0.001).astype(F)))
    lens = np.asarray([37, 64])
    for step in range(41):
        news = lens if step == 0 else np.asarray([1, 1])
        if step:
            lens = lens + 1
        starts = np.concatenate([[0], np.cumsum(news)])
        x = (rng.standard_normal((starts[-1], q + 2 * n)) * (1 + 0.1 * step)).astype(F)
        c.host.append(x[:, q:q + n], x[:, q + n:], c.table, starts, lens)
        att, logits, tok, lp, ent, ids, val = serving_step(torch, ops, c.dev, w, put(torch, x), i32(torch, starts), i32(torch, lens),
                                                          H, hd, Hk, step > 0)
        c.same()
        if step % 8 == 0:
            want, bound = attention(c.host, x[:, :q], c.table, starts, lens, H, 1 / math.sqrt(hd))
            check(torch, att, want, bound, "f32")
        lp_check(torch, logits.double().cpu().numpy(), (lp, ent, ids, val), tok.cpu().numpy(), 5, 1)
        assert torch.equal(ids[:, 0], tok) and torch.equal(lp, val[:, 0])


def test_two_graphs_on_another_stream(env):
    """Two serving steps captured side by side and replayed in turn with eager work between: every replay gives what the
    eager calls give on the same inputs."""
    torch, ops = env
    rng = np.random.default_rng(15)
    H, Hk, hd, V = 4, 2, 64, 9000
    q, n = H * hd, Hk * hd
    w = (put(torch, rng.integers(-127, 128, (V, q)).astype(np.int8)), put(torch, (rng.random(V) * 0.01 + 0.001).astype(F)))
    side = torch.cuda.Stream()
    graphs = []
    for lens in ([700, 20], [33, 1500]):
        c = Both(torch, ops, rng, [m + 8 for m in lens], Hk, hd, 64).fill(rng).send()
        qkv, ln, st = put(torch, rng.standard_normal((2, q + 2 * n)).astype(F)), i32(torch, lens), i32(torch, [0, 1, 2])
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            serving_step(torch, ops, [t.clone() for t in c.dev], w, qkv, st, ln, H, hd, Hk, True)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = serving_step(torch, ops, c.dev, w, qkv, st, ln, H, hd, Hk, True)
        graphs.append((g, out, c, qkv, st, ln))
    twin = [[t.clone() for t in c.dev] for _, _, c, _, _, _ in graphs]
    for turn in range(4):
        for i, (g, out, c, qkv, st, ln) in enumerate(graphs):
            qkv.copy_(put(torch, rng.standard_normal(qkv.shape).astype(F) * (1 + turn)))
            g.replay()
            want = serving_step(torch, ops, twin[i], w, qkv, st, ln, H, hd, Hk, True)
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b)
            for a, b in zip(c.dev, twin[i]):
                assert torch.equal(a, b)
            ln += 1


def test_graph_of_ragged_rows(env):
    """Turns and drafts captured with their appends (keys cut into parts, and whole), replayed while lengths and rows change."""
    torch, ops = env
    rng = np.random.default_rng(20)
    H, Hk, hd = 8, 2, 64
    for news, lens, width in (([5, 3], [900, 2500], 64), ([300, 180, 0], [400, 1300, 0], 64), ([700, 700], [900, 1500], 32)):
        c = Both(torch, ops, rng, lens, Hk, hd, 64, width=width).fill(rng).send()
        rows = sum(news)
        st, ln, out = i32(torch, np.concatenate([[0], np.cumsum(news)])), i32(torch, lens), None
        x = put(torch, rng.standard_normal((rows, (H + 2 * Hk) * hd)).astype(F))
        k, v, q = x[:, H * hd:(H + Hk) * hd], x[:, (H + Hk) * hd:], x[:, :H * hd]

        def turn(cache):
            ops.kv_append_block(k, v, *cache, st, ln)
            return ops.attention_block_prefill(q, *cache, st, ln, H)

        twin = [t.clone() for t in c.dev]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            turn([t.clone() for t in c.dev])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = turn(c.dev)
        for _ in range(3):
            x.copy_(put(torch, rng.standard_normal(tuple(x.shape)).astype(F)))
            g.replay()
            want = turn(twin)
            torch.cuda.synchronize()
            assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(c.dev, twin))
            ln.sub_(7).clamp_(min=0)


def test_calls_on_two_streams_at_once(env):
    """Reads of one cache from two streams, without a wait between them."""
    torch, ops = env
    rng = np.random.default_rng(21)
    H, Hk, hd = 16, 4, 128
    lens = [3000, 90, 700]
    c = Both(torch, ops, rng, lens, Hk, hd, 64).fill(rng).send()
    xs = [put(torch, rng.standard_normal((3, H * hd)).astype(F)) for _ in range(2)]
    ys = [put(torch, rng.standard_normal((120, H * hd)).astype(F)) for _ in range(2)]
    zs = [put(torch, rng.standard_normal((9, 40000)).astype(F)) for _ in range(2)]
    st = i32(torch, [0, 60, 100, 120])

    def calls(i):
        return (ops.attention_block(xs[i], *c.dev, c.lens_d, H), ops.attention_block_prefill(ys[i], *c.dev, st, c.lens_d, H),
                *ops.logprobs(zs[i], top=9)[1:])

    want = [calls(0), calls(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, calls(i)))
    torch.cuda.synchronize()
    for i, g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want[i]))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_result_in_the_query_s_place(env, dtype):
    """The C entry points with out = q, whose rows lie apart: the same values as in a place of their own, and what lies between
    the rows as it was."""
    torch, ops = env
    from t2r_amd import abi
    rng = np.random.default_rng(22)
    H, Hk, hd, block = 8, 2, 64, 64
    code = {"f32": abi.T2R_F32, "bf16": abi.T2R_BF16}[dtype]
    s = torch.cuda.current_stream().cuda_stream
    for lens, news in (([300, 1], None), ([5000, 700], None), ([300, 90], [300, 17]), ([4000, 900], [6, 2]), ([2000, 0, 40], [1500, 0, 3])):
        c = Both(torch, ops, rng, lens, Hk, hd, block).fill(rng).send()
        rows, B = sum(news or [1] * len(lens)), len(lens)
        _, t = rounded(torch, rng.standard_normal((rows, H * hd + 8)), dtype)
        q = t[:, :H * hd]
        st = i32(torch, np.concatenate([[0], np.cumsum(news)])) if news else None
        want = ops.attention_block_prefill(q, *c.dev, st, c.lens_d, H) if news else ops.attention_block(q, *c.dev, c.lens_d, H)
        kc, vc, ks, vs, table = c.dev
        n, width = kc.shape[0], table.shape[1]
        need = abi.load().t2r_attn_blk_workspace_bytes(B, rows if news else 0, H, Hk, hd, block, width, code)
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda:0")
        beside = t[:, H * hd:].clone()
        head = (t.data_ptr(), code, t.stride(0), kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr(), n, block, Hk, hd, table.data_ptr(), width)
        tail = (H, 1 / math.sqrt(hd), t.data_ptr(), t.stride(0), ws.data_ptr(), need, s)
        if news:
            abi.call("t2r_attn_blk_prefill", *head, st.data_ptr(), c.lens_d.data_ptr(), B, rows, *tail)
        else:
            abi.call("t2r_attn_blk_decode", *head, c.lens_d.data_ptr(), B, *tail)
        torch.cuda.synchronize()
        assert torch.equal(t[:, :H * hd], want) and torch.equal(t[:, H * hd:], beside)


def test_same_bits_every_time(env):
    torch, ops = env
    rng = np.random.default_rng(16)
    H, Hk, hd = 16, 4, 128
    lens = [1500, 90, 700]
    c = Both(torch, ops, rng, lens, Hk, hd, 64, width=128).fill(rng).send()
    x = put(torch, rng.standard_normal((3, H * hd)).astype(F))
    y = put(torch, rng.standard_normal((120, H * hd)).astype(F))
    st = i32(torch, [0, 60, 100, 120])
    z = put(torch, rng.standard_normal((9, 40000)).astype(F))
    first = (ops.attention_block(x, *c.dev, c.lens_d, H), ops.attention_block_prefill(y, *c.dev, st, c.lens_d, H), *ops.logprobs(z, top=9)[1:])
    for _ in range(5):
        again = (ops.attention_block(x, *c.dev, c.lens_d, H), ops.attention_block_prefill(y, *c.dev, st, c.lens_d, H), *ops.logprobs(z, top=9)[1:])
        for a, b in zip(first, again):
            assert torch.equal(a, b)


def test_empty_calls(env):
    torch, ops = env
    c = ops.block_cache(4, 2, 32, 16)
    table, st, ln = i32(torch, [[0, 1]]), i32(torch, [0, 0]), i32(torch, [0])
    x = torch.empty((0, 64), device="cuda:0")
    ops.kv_append_block(x, x, *c, table, st, ln)
    assert ops.attention_block_prefill(x, *c, table, st, ln, 2).shape == (0, 64)
    assert ops.kv_read_block(*c, table, st, ln, 0)[0].shape == (0, 64)
    assert ops.attention_block(x, *c, table[:0], ln[:0], 2).shape == (0, 64)
    assert ops.logprobs(torch.empty((0, 50), device="cuda:0"), top=3)[2].shape == (0, 3)
