"""Attention over the block-scaled cache (t2r_amd.ops) at lengths and mixes that its other tests do not reach: many parts of a
row, rows without a place beside long ones, prompts and single tokens in one call, batches of mostly idle sequences."""
import math

import numpy as np
import pytest

from blockref import attention
from test_gpu_block import Both, check, env, i32, rounded  # noqa: F401 (env is the fixture)

pytestmark = pytest.mark.gpu
W16 = 2.0 ** -11                                                          # of a weight that is one fp16 number


def run_rows(env, H, Hk, hd, block, news, lens, width, dtype, only, seed, spread=1.0):
    torch, ops = env
    rng = np.random.default_rng(seed)
    c = Both(torch, ops, rng, lens, Hk, hd, block, width=width).fill(rng, spread=spread).send()
    starts = np.concatenate([[0], np.cumsum(news)])
    x, t = rounded(torch, rng.standard_normal((starts[-1], H * hd)), dtype)
    got = ops.attention_block_prefill(t, *c.dev, i32(torch, starts), c.lens_d, H)
    want, bound = attention(c.host, x, c.table, starts, lens, H, 1 / math.sqrt(hd), 0 if dtype == "f32" else W16, only=only)
    check(torch, got, want, bound, dtype)
    return got


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("n", [16640, 40001])
def test_step_of_more_than_64_parts(env, n, dtype):
    """One sequence of one KV head in a wide table, in parts of 256 keys: the join takes them 64 at a time."""
    torch, ops = env
    rng = np.random.default_rng(n)
    H, Hk, hd = 4, 1, 32
    c = Both(torch, ops, rng, [n], Hk, hd, 128, width=384).fill(rng, spread=1.5).send()
    x, t = rounded(torch, rng.standard_normal((1, H * hd)), dtype)
    want, bound = attention(c.host, x, c.table, [0, 1], [n], H, 1 / math.sqrt(hd), 0 if dtype == "f32" else W16)
    check(torch, ops.attention_block(t, *c.dev, c.lens_d, H), want, bound, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_drafts_of_more_than_64_parts(env, dtype):
    """Rows of one sequence over more than 64 parts of 512 keys."""
    run_rows(env, 4, 1, 32, 128, [5], [40001], 400, dtype, None, 71, 1.5)


@pytest.mark.parametrize("H,Hk,hd,block,news,lens,width", [
    (8, 2, 64, 64, [9, 4], [7, 3000], 64),                                 # few rows, in parts
    (32, 8, 64, 64, [40, 200], [33, 3000], 64),                            # turns, in parts
])
def test_rows_without_a_place_beside_long_ones(env, H, Hk, hd, block, news, lens, width):
    """Rows below position 0 give NaN in a call whose long sequence is cut into parts; the others are what they are."""
    torch, _ = env
    got = run_rows(env, H, Hk, hd, block, news, lens, width, "f32", set(range(news[0])) | {news[0], sum(news) - 1}, 72)
    lost = news[0] - lens[0]
    assert torch.isnan(got[:lost]).all() and torch.isfinite(got[lost:]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_prompt_and_single_tokens_in_one_call(env, dtype):
    """A serving step's ragged batch: eleven conversations with a token each, some long, and a prompt among them."""
    lens = [1, 700, 2600, 64, 65, 5, 300, 1999, 31, 128, 640, 17]
    news = [1] * 6 + [300] + [1] * 5
    run_rows(env, 16, 4, 64, 64, news, lens, 64, dtype, {*range(6), 6, 7, 150, 304, 305, *range(306, 311)}, 73)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_prompt_among_idle_sequences(env, dtype):
    """A prompt in a batch of 100 slots, the others idle or empty."""
    lens, news = [0] * 100, [0] * 100
    lens[37], news[37] = 450, 400
    lens[99], lens[2] = 77, 12
    run_rows(env, 8, 2, 64, 32, news, lens, 40, dtype, {0, 1, 7, 8, 200, 398, 399}, 74)


@pytest.mark.parametrize("H,Hk,hd,block,news,lens,width", [
    (32, 8, 64, 64, [548], [4500], 128),                                   # late turns in long caches
    (16, 8, 128, 32, [300, 0, 251], [3300, 40, 2900], 256),
    (32, 32, 64, 64, [700, 400], [4500, 2100], None),                      # tiles over several segments
    (32, 32, 128, 64, [700, 400], [4500, 2100], None),
])
def test_long_caches_in_fp16(env, H, Hk, hd, block, news, lens, width):
    run_rows(env, H, Hk, hd, block, news, lens, width, "f16", {0, 15, 333, news[0] - 1, sum(news) - 1}, 75, 1.5)
