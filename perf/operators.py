"""What the block-scaled KV cache, the attention over it and the token log probabilities are measured on.

The cache holds int8 codes in blocks of `block` tokens, with one float32 scale for each block and KV head, and a table
that says which block of the pool holds which tokens of a sequence:

    kc [blocks, Hk, block, hd] int8     key codes              ks [blocks, Hk] float32
    vc [blocks, Hk, hd, block] int8     value codes            vs [blocks, Hk] float32
    table [B, width] int32              position p of sequence b lies in block table[b, p // block], slot p % block

Rows of several sequences come as one ragged batch: those of sequence b are starts[b] .. starts[b + 1] - 1, and the last
of them stands at position lens[b] - 1. `own` calls t2r_amd.ops; the plain forms are elementary torch operations.
"""
import math

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one token of each of 16 conversations enters the cache (the heads of the 1B model); latency counts
        dict(name="append-step-16", kind="append", B=16, H=32, Hk=8, hd=64, block=64, lo=33, hi=1999, new=1, cap=2048, dtype="f32"),
        # the longest prompt of a 2048-position cache enters it in one call
        dict(name="append-prompt-2032", kind="append", B=1, H=16, Hk=8, hd=128, block=64, lo=2032, hi=2032, new=2032, cap=2048, dtype="f32"),
        # further turns of five conversations of odd lengths, from a host that keeps its activations in 16 bits
        dict(name="append-turns-bf16", kind="append", B=5, H=9, Hk=3, hd=64, block=32, lo=411, hi=3001, new=333, cap=4096, dtype="bf16"),
        # the smallest call: one token of a small model early in a conversation. Launches count.
        dict(name="step-1-short", kind="step", B=1, H=9, Hk=3, hd=64, block=64, lo=96, hi=96, cap=2048, dtype="f32"),
        # one token late in a long conversation: few rows, long caches
        dict(name="step-1-long", kind="step", B=1, H=32, Hk=8, hd=64, block=64, lo=8101, hi=8101, cap=8192, dtype="f32"),
        # a full serving step over long caches: the cache's bytes count
        dict(name="step-32-long", kind="step", B=32, H=16, Hk=8, hd=128, block=64, lo=1021, hi=8192, cap=8192, dtype="f32"),
        # many short conversations of the smallest model, no shared heads, small blocks, 16-bit activations
        dict(name="step-24-bf16", kind="step", B=24, H=6, Hk=6, hd=48, block=16, lo=1, hi=255, cap=256, dtype="bf16"),
        # the longest prompt in one call
        dict(name="prompt-2032", kind="prompt", B=1, H=16, Hk=8, hd=128, block=64, lo=2032, hi=2032, new=2032, cap=2048, dtype="f32"),
        # prompts and further turns of seven conversations, 16-bit activations
        dict(name="prompt-turns-bf16", kind="prompt", B=7, H=32, Hk=8, hd=64, block=64, lo=190, hi=3100, new=701, cap=4096, dtype="bf16"),
        # eight drafted tokens of each of four long conversations are looked at in one call
        dict(name="prompt-drafts", kind="prompt", B=4, H=32, Hk=8, hd=64, block=64, lo=5003, hi=8100, new=8, cap=8192, dtype="f32"),
        # the answer tokens of a serving step, with the alternatives that an API returns
        dict(name="logprobs-step-16", kind="logprobs", rows=16, vocab=128256, top=20, dtype="f32"),
        # a prompt is scored whole: an odd vocabulary (rows off every alignment), 16-bit logits
        dict(name="logprobs-prompt-bf16", kind="logprobs", rows=2032, vocab=49155, top=5, dtype="bf16"),
    ]


HEADS = [(6, 6, 48), (9, 3, 64), (16, 8, 128), (32, 8, 64), (16, 8, 64), (8, 1, 64), (12, 4, 80), (10, 5, 96), (4, 2, 16),
         (24, 2, 128), (7, 7, 32)]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "append", "step", "step", "step", "prompt", "prompt", "prompt", "logprobs", "logprobs"])
    dtype = rng.choice(["f32", "f32", "bf16", "f16"])
    if kind == "logprobs":
        vocab = _log(rng, 61, 151936)
        return dict(kind=kind, rows=_log(rng, 1, max(1, min(2032, 50_000_000 // vocab))), vocab=vocab, top=rng.choice([0, 1, 5, 20]),
                    dtype=dtype)
    H, Hk, hd = rng.choice(HEADS)
    block = rng.choice([16, 32, 64, 64, 128])
    cap = rng.choice([256, 1024, 2048, 4096, 8192])
    c = dict(kind=kind, H=H, Hk=Hk, hd=hd, block=block, cap=cap, dtype=dtype)
    if kind == "step":
        lo = _log(rng, 1, cap)
        return dict(c, B=_log(rng, 1, 32), lo=lo, hi=_log(rng, lo, cap))
    new = _log(rng, 1, min(cap, 2032))
    lo = _log(rng, new, cap)
    hi = _log(rng, lo, cap)
    B = _log(rng, 1, 16)
    most = 2_000_000 if kind == "append" else 8_000_000_000     # values a cache takes in; multiply-adds of the scores
    one = new * Hk * hd if kind == "append" else new * hi * H * hd
    if one > most:                                            # never more than the largest listed case
        new = max(1, int(new * most / one))
        one = most
    return dict(c, B=max(1, min(B, most // one)), lo=max(lo, new), hi=max(hi, new), new=new)


# ------------------------------------------------------------------ inputs
def _lens(case):
    """The sequences' lengths, spread from lo to hi."""
    B = case["B"]
    if B == 1:
        return [case["hi"]]
    return [case["lo"] + (case["hi"] - case["lo"]) * ((7 * b + B // 2) % B) // (B - 1) if math.gcd(7, B) == 1 else
            case["lo"] + (case["hi"] - case["lo"]) * b // (B - 1) for b in range(B)]


def _news(case):
    """How many of each sequence's rows are new: between a third of `new` and all of it."""
    if case["kind"] == "step":
        return [1] * case["B"]
    return [max(1, case["new"] - case["new"] * ((5 * b) % 8) // 12) for b in range(case["B"])]


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(1 + int(seed))


def _starts(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    g = _gen(seed)
    dt = TYPES[case["dtype"]]
    if case["kind"] == "logprobs":
        rows, V = case["rows"], case["vocab"]
        x = torch.randn((rows, V), generator=g, device=DEV).mul_(2.2)       # a body and a few favourites, as a model's logits
        fav = torch.randint(0, V, (rows, 6), generator=g, device=DEV)
        x.scatter_add_(1, fav, torch.rand((rows, 6), generator=g, device=DEV) * 12)
        tok = torch.where(torch.rand(rows, generator=g, device=DEV) < 0.7, fav[:, 0],
                          torch.randint(0, V, (rows,), generator=g, device=DEV)).to(torch.int32)
        return dict(case=case, logits=x.to(dt), tokens=tok)
    B, H, Hk, hd, bs = (case[k] for k in ("B", "H", "Hk", "hd", "block"))
    lens, news = _lens(case), _news(case)
    width = -(-case["cap"] // bs)
    used = [-(-n // bs) for n in lens]
    pool = sum(used) + 3
    order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)    # a pool that has seen sequences come and go
    table = torch.full((B, width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n

    def codes(*shape):
        return torch.randn(shape, generator=g, device=DEV).mul_(127 / 3.6).round_().clamp_(-127, 127).to(torch.int8)

    def scales():
        return (torch.randn((pool, Hk), generator=g, device=DEV) * 0.3).exp_() * (3.6 / 127)

    st = dict(case=case, kc=codes(pool, Hk, bs, hd), vc=codes(pool, Hk, hd, bs), ks=scales(), vs=scales(), table=table,
              lens=_i32(lens))
    rows = sum(news)
    # the rows as a linear layer leaves them: q | k | v side by side
    st["qkv"] = torch.randn((rows, (H + 2 * Hk) * hd), generator=g, device=DEV).to(dt)
    st["starts"] = _i32(_starts(news))
    if case["kind"] == "append":
        # every block that a row enters is looked at whole: its older rows may have moved to a larger scale
        first = [(n - k) // bs * bs for n, k in zip(lens, news)]
        span = [n - f for n, f in zip(lens, first)]
        st["span_starts"], st["span_rows"] = _i32(_starts(span)), sum(span)
        st["touched"] = torch.cat([table[b, f // bs:u] for b, (f, u) in enumerate(zip(first, used))]).long()
    return st


# ------------------------------------------------------------------ one pass
def run(st):
    kind = st["case"]["kind"]
    if kind == "logprobs":
        return _own_logprobs(st) if own else _plain_logprobs(st)
    if kind == "append":
        return _own_append(st) if own else _plain_append(st)
    return _own_attention(st) if own else _plain_attention(st)


def _own_logprobs(st):
    from t2r_amd import ops
    lp, ent, ids, top = ops.logprobs(st["logits"], st["tokens"], top=st["case"]["top"])
    return [lp, ent, ids, top]


def _own_append(st):
    from t2r_amd import ops
    c = st["case"]
    q, kv = c["H"] * c["hd"], c["Hk"] * c["hd"]
    x, cache = st["qkv"], (st["kc"], st["vc"], st["ks"], st["vs"], st["table"])
    ops.kv_append_block(x[:, q:q + kv], x[:, q + kv:], *cache, st["starts"], st["lens"])
    k, v = ops.kv_read_block(*cache, st["span_starts"], st["lens"], st["span_rows"])
    return [k, v, st["ks"], st["vs"]]


def _own_attention(st):
    from t2r_amd import ops
    c = st["case"]
    q, cache = st["qkv"][:, :c["H"] * c["hd"]], (st["kc"], st["vc"], st["ks"], st["vs"], st["table"])
    if c["kind"] == "step":
        return [ops.attention_block(q, *cache, st["lens"], c["H"])]
    return [ops.attention_block_prefill(q, *cache, st["starts"], st["lens"], c["H"])]


# ------------------------------------------------------------------ the plain forms
def _plain_logprobs(st):
    x, top = st["logits"].float(), st["case"]["top"]
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    l = e.sum(1, keepdim=True)
    lse = m + torch.log(l)
    lp = x.gather(1, st["tokens"].long()[:, None]) - lse
    ent = torch.log(l) - (e * (x - m)).sum(1, keepdim=True) / l
    val, ids = torch.sort(x, dim=1, descending=True, stable=True)
    return [lp[:, 0], ent[:, 0], ids[:, :top].to(torch.int32), val[:, :top] - lse]


def _row_places(starts, lens, rows):
    """The sequence and the position of each row."""
    r = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(starts.long(), r, right=True) - 1
    return seq, lens.long()[seq] - starts.long()[seq + 1] + r


def _plain_append(st):
    c = st["case"]
    H, Hk, hd, bs = (c[k] for k in ("H", "Hk", "hd", "block"))
    rows = st["qkv"].shape[0]
    seq, pos = _row_places(st["starts"], st["lens"], rows)
    blk, slot = st["table"].long()[seq, pos // bs], pos % bs
    first = torch.full((st["ks"].shape[0],), bs, device=DEV).index_reduce_(0, blk, slot, "amin")
    t = st["touched"]
    x = st["qkv"][:, H * hd:].float().view(rows, 2, Hk, hd)
    for i, (code, scale, flip) in enumerate(((st["kc"], st["ks"], False), (st["vc"], st["vs"], True))):
        new = torch.zeros_like(scale).index_reduce_(0, blk, x[:, i].abs().amax(-1), "amax")
        new = (new.double() / 127).float()                     # (torch takes a float32 quotient by a number as a product)
        s = torch.where(first[t, None] > 0, torch.maximum(scale[t], new[t]), new[t])
        tile = code[t].transpose(2, 3) if flip else code[t]                          # [blocks, Hk, block, hd]
        moved = (tile.double() * scale[t].double()[..., None, None] / s.double()[..., None, None]).round()
        old = torch.arange(bs, device=DEV)[None, :] < first[t, None]
        tile = torch.where(old[:, None, :, None], moved, tile.double()).to(torch.int8)      # (slots behind the rows stay)
        code[t] = tile.transpose(2, 3).contiguous() if flip else tile
        scale[t] = s
        # (64 bits: a quotient next to a half is rounded to the side that it is on)
        y = (x[:, i].double() / scale[blk].double()[..., None]).nan_to_num_(0.0).round().clamp_(-127, 127).to(torch.int8)
        if flip:
            code[blk, :, :, slot] = y
        else:
            code[blk, :, slot] = y
    seq, pos = _row_places(st["span_starts"], st["lens"], st["span_rows"])
    blk, slot = st["table"].long()[seq, pos // bs], pos % bs
    k = st["kc"][blk, :, slot].float() * st["ks"][blk][..., None]
    v = st["vc"][blk, :, :, slot].float() * st["vs"][blk][..., None]
    return [k.reshape(-1, Hk * hd), v.reshape(-1, Hk * hd), st["ks"], st["vs"]]


def _plain_attention(st):
    c = st["case"]
    B, H, Hk, hd, bs = (c[k] for k in ("B", "H", "Hk", "hd", "block"))
    rows, most = st["qkv"].shape[0], max(_news(c))
    pages = -(-max(_lens(c)) // bs)
    tab = st["table"][:, :pages].long().clamp_min(0)
    # every sequence's keys and values side by side, [B, Hk, positions, hd]
    k = (st["kc"][tab].float() * st["ks"][tab][..., None, None]).transpose(1, 2).reshape(B, Hk, -1, hd)
    v = (st["vc"][tab].float() * st["vs"][tab][..., None, None]).permute(0, 2, 1, 4, 3).reshape(B, Hk, -1, hd)
    seq, pos = _row_places(st["starts"], st["lens"], rows)
    i = torch.arange(rows, device=DEV) - st["starts"].long()[seq]
    q = torch.zeros((B, most, H, hd), device=DEV)
    q[seq, i] = st["qkv"][:, :H * hd].float().view(rows, H, hd)
    at = torch.full((B, most), 0, device=DEV)
    at[seq, i] = pos
    q = q.view(B, most, Hk, H // Hk, hd).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, hd)     # rows of a KV head's heads
    s = torch.matmul(q, k.transpose(2, 3).contiguous()).view(B, Hk, H // Hk, most, -1) * (1 / math.sqrt(hd))
    s = s.masked_fill_(torch.arange(s.shape[-1], device=DEV) > at[:, None, None, :, None], float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).view(B, Hk, -1, p.shape[-1])
    o = torch.matmul(p, v).view(B, Hk, H // Hk, most, hd).permute(0, 3, 1, 2, 4)
    return [o[seq, i].reshape(rows, H * hd).to(st["qkv"].dtype)]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * es + case["rows"] * (12 + 8 * case["top"]), "flops": 6 * n}
    lens, news = _lens(case), _news(case)
    q, kv, bs = case["H"] * case["hd"], case["Hk"] * case["hd"], case["block"]
    if case["kind"] == "append":
        span = sum(n - (n - k) // bs * bs for n, k in zip(lens, news))
        return {"bytes": 2 * kv * (sum(news) * (es + 1) + span * (1 + 4)), "flops": 2 * kv * (4 * sum(news) + span)}
    keys = sum((n - k + i + 1) for n, k in zip(lens, news) for i in range(k))
    return {"bytes": 2 * kv * sum(lens) + 2 * es * sum(news) * q, "flops": 4 * keys * q}


# ------------------------------------------------------------------ the same in float64
def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "logprobs":
        return _exact_logprobs(st)
    if case["kind"] == "append":
        return _exact_append(st)
    return _exact_attention(st)


def _exact_logprobs(st):
    lp, ent, top = [], [], []
    for x, t in zip(st["logits"], st["tokens"].tolist()):
        y = x.double()
        z = torch.logsumexp(y, 0)
        p = torch.exp(y - z)
        lp.append(y[t] - z)
        ent.append(z - (p * y).sum())
        top.append(torch.topk(y, st["case"]["top"])[0] - z)
    return [torch.stack(lp), torch.stack(ent), None, torch.stack(top)]


def _exact_append(st):
    c = st["case"]
    H, Hk, hd, bs = (c[k] for k in ("H", "Hk", "hd", "block"))
    at = st["starts"].tolist()
    new = st["qkv"][:, H * hd:].double().reshape(-1, 2, Hk, hd)
    table = st["table"].tolist()
    scale = [st["ks"].double(), st["vs"].double()]
    code = [st["kc"].double(), st["vc"].double().transpose(2, 3).contiguous()]
    out = [[], []]
    for b, n in enumerate(st["lens"].tolist()):
        p0 = n - (at[b + 1] - at[b])
        for j in range(p0 // bs, -(-n // bs)):
            lo, hi, blk = max(p0 - j * bs, 0), min(n - j * bs, bs), table[b][j]
            r = at[b] + j * bs + lo - p0
            for i in range(2):
                x = new[r:r + hi - lo, i].transpose(0, 1)                   # [Hk, rows, hd]
                s = (x.abs().amax((1, 2)) / 127).float().double()          # a scale is a float32 number
                if lo:
                    was = scale[i][blk]
                    s = torch.maximum(was, s)
                    code[i][blk, :, :lo] = (code[i][blk, :, :lo] * was[:, None, None] / s[:, None, None]).round()
                code[i][blk, :, lo:hi] = (x / s[:, None, None]).round().clamp(-127, 127)
                scale[i][blk] = s
                out[i].append((code[i][blk, :, :hi] * s[:, None, None]).transpose(0, 1).reshape(hi, Hk * hd))
    return [torch.cat(out[0]), torch.cat(out[1]), scale[0], scale[1]]


def _exact_attention(st):
    c = st["case"]
    H, Hk, hd, bs = (c[k] for k in ("H", "Hk", "hd", "block"))
    at, out = st["starts"].tolist(), []
    for b, n in enumerate(st["lens"].tolist()):
        pages = st["table"][b, :-(-n // bs)].long()
        k = (st["kc"][pages].double() * st["ks"][pages].double()[..., None, None]).transpose(0, 1).reshape(Hk, -1, hd)[:, :n]
        v = (st["vc"][pages].double() * st["vs"][pages].double()[..., None, None]).permute(1, 0, 3, 2).reshape(Hk, -1, hd)[:, :n]
        q = st["qkv"][at[b]:at[b + 1], :H * hd].double().view(-1, H, hd)
        seen = torch.arange(n, device=DEV)[None] <= torch.arange(n - q.shape[0], n, device=DEV)[:, None]
        o = torch.empty_like(q)
        for h in range(H):
            s = (q[:, h] @ k[h * Hk // H].T / math.sqrt(hd)).masked_fill(~seen, float("-inf"))
            o[:, h] = torch.softmax(s, -1) @ v[h * Hk // H]
        out.append(o.reshape(-1, H * hd))
    return [torch.cat(out)]
