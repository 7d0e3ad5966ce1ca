"""Op-level calls on torch device tensors: one C-ABI call (one or two HIP launches) per piece of
the reference's token list (llm/compile_model.py:147-349), each step for step the DeviceModel
method it names (llm/ref_model.py:191-255). Inputs must be contiguous tensors on a HIP device
with the dtypes below; outputs are allocated here (the C-ABI itself never allocates).

The calls at the end (the block-scaled KV cache, the attention over it, log probabilities) have no counterpart in the
reference. They take float32, bfloat16 or float16 rows that may lie apart (columns of a larger matrix), run on their
tensors' own device and use that device's current stream."""
import functools
import math

import torch

from . import abi

I8, I32, F32 = torch.int8, torch.int32, torch.float32


def _dev(*ts):
    for t in ts:
        if t is not None and (not t.is_cuda or not t.is_contiguous()):
            raise ValueError("op arguments must be contiguous tensors on a HIP device")


def _s():
    return abi.stream_ptr()


def _u32(t):
    return t.view(torch.int32) if t.dtype == torch.float32 else t


def sfu(fn, x_bits):
    """fn 'exp' | 'recip' | 'rsqrt' | 'abs' on fp32 bit patterns (int32 tensor) -> bit patterns."""
    _dev(x_bits)
    code = {"exp": 0, "recip": 1, "rsqrt": 2, "abs": 3}[fn]
    y = torch.empty_like(x_bits)
    abi.call("t2r_sfu", code, abi.ptr(x_bits), abi.ptr(y), x_bits.numel(), _s())
    return y


def sfu_check(fn, first=0, count=1 << 32):
    """Inputs [first, first + count) through the datapath SFU and the literal FTZ sequence; returns
    (number of differing results, smallest differing input or None). 'exp_np': the softmax's EXP,
    checked against EXP on its domain (x <= 0 and NaN); 'recip_ge1': the gates' RECIP, against RECIP
    on its domain (x >= 1 and NaN); 'exp_sm': the softmax's EXP under a finite maximum, against EXP
    on its domain (x <= 0); 'exp_g' / 'recip_g1': the gates' pair-table EXP (x not NaN) and RECIP
    (x >= 1, not NaN), against EXP and RECIP; other inputs skipped."""
    code = {"exp": 0, "recip": 1, "rsqrt": 2, "exp_np": 3, "recip_ge1": 4, "exp_sm": 5, "exp_g": 6, "recip_g1": 7}[fn]
    out = torch.empty(2, dtype=torch.int32, device="cuda")
    abi.call("t2r_sfu_check", code, first, count, abi.ptr(out), _s())
    n, lo = (int(v) & 0xFFFFFFFF for v in out.cpu().tolist())
    return n, (None if n == 0 else lo)


def fp32_op(op, a_bits, b_bits):
    """The fp32 primitives on bit patterns: 'add', 'sub', 'mul', 'ldexp', 'floor', 'to_i8', 'from_int',
    'ieee_mul', 'ieee_add' (see include/t2r.h t2r_fp32_op)."""
    _dev(a_bits, b_bits)
    code = ["add", "sub", "mul", "ldexp", "floor", "to_i8", "from_int", "ieee_mul", "ieee_add"].index(op)
    y = torch.empty_like(a_bits)
    abi.call("t2r_fp32_op", code, abi.ptr(a_bits), abi.ptr(b_bits), abi.ptr(y), a_bits.numel(), _s())
    return y


def requant(r, scale, shift, zp, lo, hi):
    _dev(r)
    out = torch.empty(r.shape, dtype=I8, device=r.device)
    abi.call("t2r_requant", abi.ptr(r), r.numel(), int(scale), int(shift), int(zp), int(lo), int(hi), abi.ptr(out), _s())
    return out


def embed(emb_q, emb_s, tokens):
    _dev(emb_q, emb_s, tokens)
    V, d = emb_q.shape
    x = torch.empty((tokens.numel(), d), dtype=F32, device=emb_q.device)
    abi.call("t2r_embed", abi.ptr(emb_q), abi.ptr(emb_s), abi.ptr(tokens), tokens.numel(), d, V, abi.ptr(x), None, _s())
    return x


def rmsnorm(x, g, eps, D):
    _dev(x, g)
    out = torch.empty_like(x)
    n = x.shape[-1]
    abi.call("t2r_rmsnorm", abi.ptr(x), abi.ptr(g), x.numel() // n, n, float(eps), int(D), abi.ptr(out), _s())
    return out


def quant_act(x):
    _dev(x)
    n = x.shape[-1]
    rows = x.numel() // n
    xq = torch.empty(x.shape, dtype=I8, device=x.device)
    s = torch.empty(x.shape[:-1] if x.dim() > 1 else (1,), dtype=F32, device=x.device)
    abi.call("t2r_quant_act", abi.ptr(x), rows, n, abi.ptr(xq), abi.ptr(s), _s())
    return xq, s


def linear(w, s_w, xq, s_x, residual=None, acc=False):
    """W8A8 linear of rows xq [M, K] (or [K]); returns y (and the int32 accumulators with acc=True)."""
    _dev(w, s_w, xq, s_x, residual)
    N, K = w.shape
    M = xq.numel() // K
    y = torch.empty((M, N) if xq.dim() > 1 else (N,), dtype=F32, device=w.device)
    a = torch.empty(y.shape, dtype=I32, device=w.device) if acc else None
    name = "t2r_gemv_w8a8" if xq.dim() == 1 else "t2r_gemm_w8a8"
    args = [abi.ptr(w), abi.ptr(s_w), abi.ptr(xq), abi.ptr(s_x)] + ([] if xq.dim() == 1 else [M]) + \
        [N, K, abi.ptr(y), abi.ptr(a), abi.ptr(residual), _s()]
    abi.call(name, *args)
    return (y, a) if acc else y


def rope(v, cos_t, sin_t, pos):
    """RoPE of rows v [rows, n] in place (heads of head_dim = 2 * cos_t.shape[1])."""
    _dev(v, cos_t, sin_t, pos)
    n = v.shape[-1]
    abi.call("t2r_rope", abi.ptr(v), abi.ptr(cos_t), abi.ptr(sin_t), abi.ptr(pos), v.numel() // n, n,
             cos_t.shape[1], cos_t.shape[0], _s())
    return v


def kv_append(k, v, inv_sk, inv_sv, kc, vc, pos):
    _dev(k, v, kc, vc, pos)
    kv = kc.shape[-1]
    abi.call("t2r_kv_append", abi.ptr(k), abi.ptr(v), float(inv_sk), float(inv_sv), abi.ptr(kc), abi.ptr(vc),
             abi.ptr(pos), k.numel() // kv, kv, kc.shape[0], _s())


def kv_append_ch(k, v, inv_sk, inv_sv, kc, vc, pos):
    """KV append with per-channel inverse scales: inv_sk / inv_sv are [kv_dim] device tensors or scalars."""
    _dev(k, v, kc, vc, pos)
    kv = kc.shape[-1]
    vec = lambda x: abi.ptr(x) if isinstance(x, torch.Tensor) else None
    sca = lambda x: 0.0 if isinstance(x, torch.Tensor) else float(x)
    abi.call("t2r_kv_append_ch", abi.ptr(k), abi.ptr(v), sca(inv_sk), sca(inv_sv), vec(inv_sk), vec(inv_sv),
             abi.ptr(kc), abi.ptr(vc), abi.ptr(pos), k.numel() // kv, kv, kc.shape[0], _s())


def attention(q, kc, vc, pos, H, Hk, a_k, a_v, D):
    """Attention of rows q [rows, H * hd] at positions pos over the int8 caches [S, Hk * hd]."""
    _dev(q, kc, vc, pos)
    hd = q.shape[-1] // H
    rows = q.numel() // q.shape[-1]
    att = torch.empty_like(q)
    abi.call("t2r_attn_decode", abi.ptr(q), abi.ptr(kc), abi.ptr(vc), abi.ptr(pos), rows, H, Hk, hd, kc.shape[0],
             float(a_k), float(a_v), int(D), abi.ptr(att), _s())
    return att


def attention_opt(q, kc, vc, pos, H, Hk, a_k, a_v, D, qsum=False, ch_sk=None, ch_av=None):
    """attention() with the HF path's options: qsum normalisation, K per channel (ch_sk [Hk * hd]: q
    multiplied before its quantisation), V per channel (ch_av [Hk * hd] in place of a_v)."""
    _dev(q, kc, vc, pos)
    hd = q.shape[-1] // H
    rows = q.numel() // q.shape[-1]
    att = torch.empty_like(q)
    abi.call("t2r_attn_decode_opt", abi.ptr(q), abi.ptr(kc), abi.ptr(vc), abi.ptr(pos), rows, H, Hk, hd,
             kc.shape[0], float(a_k), float(a_v), int(D), abi.T2R_ATTN_QSUM if qsum else 0, abi.ptr(ch_sk),
             abi.ptr(ch_av), abi.ptr(att), _s())
    return att


def attention_prefill(q, kc, vc, pos, H, Hk, a_k, a_v, D, qsum=False, ch_sk=None, ch_av=None):
    """Prefill attention of prompt rows q [M, H * hd] at positions pos [M] (t2r_attn_prefill): each row
    as attention_opt computes it, the rows on the multi-row kernel where the shape allows."""
    _dev(q, kc, vc, pos)
    hd = q.shape[-1] // H
    rows = q.numel() // q.shape[-1]
    att = torch.empty_like(q)
    abi.call("t2r_attn_prefill", abi.ptr(q), abi.ptr(kc), abi.ptr(vc), abi.ptr(pos), rows, H, Hk, hd,
             kc.shape[0], float(a_k), float(a_v), int(D), abi.T2R_ATTN_QSUM if qsum else 0, abi.ptr(ch_sk),
             abi.ptr(ch_av), abi.ptr(att), _s())
    return att


def swiglu(w1, s_w1, w3, s_w3, xq, s_x):
    _dev(w1, s_w1, w3, s_w3, xq, s_x)
    F_, K = w1.shape
    u = torch.empty(F_, dtype=F32, device=w1.device)
    hq = torch.empty(F_, dtype=I8, device=w1.device)
    s_h = torch.empty(1, dtype=F32, device=w1.device)
    abi.call("t2r_swiglu_w8a8", abi.ptr(w1), abi.ptr(s_w1), abi.ptr(w3), abi.ptr(s_w3), abi.ptr(xq), abi.ptr(s_x),
             F_, K, abi.ptr(u), abi.ptr(hq), abi.ptr(s_h), _s())
    return u, hq, s_h


def gated_ffn(act, w1, s_w1, w3, s_w3, xq, s_x):
    """The gated up-projection with gate activation act ("silu" or "gelu_tanh"), then quant_act."""
    _dev(w1, s_w1, w3, s_w3, xq, s_x)
    F_, K = w1.shape
    u = torch.empty(F_, dtype=F32, device=w1.device)
    hq = torch.empty(F_, dtype=I8, device=w1.device)
    s_h = torch.empty(1, dtype=F32, device=w1.device)
    code = {"silu": 0, "gelu_tanh": 1}[act]
    abi.call("t2r_gated_ffn_w8a8", code, abi.ptr(w1), abi.ptr(s_w1), abi.ptr(w3), abi.ptr(s_w3), abi.ptr(xq),
             abi.ptr(s_x), F_, K, abi.ptr(u), abi.ptr(hq), abi.ptr(s_h), _s())
    return u, hq, s_h


def moe_route(scores, k, D):
    _dev(scores)
    E = scores.shape[-1]
    rows = scores.numel() // E
    ids = torch.empty((rows, k), dtype=I32, device=scores.device)
    w = torch.empty((rows, k), dtype=F32, device=scores.device)
    abi.call("t2r_moe_route", abi.ptr(scores), rows, E, int(k), int(D), abi.ptr(ids), abi.ptr(w), _s())
    return ids, w


def argmax(x):
    _dev(x)
    n = x.shape[-1]
    rows = x.numel() // n
    idx = torch.empty(rows, dtype=I32, device=x.device)
    abi.call("t2r_argmax", abi.ptr(x), rows, n, abi.ptr(idx), _s())
    return idx


# ------------------------------------------------------------------ the block-scaled KV cache
_DTYPES = {torch.float32: abi.T2R_F32, torch.bfloat16: abi.T2R_BF16, torch.float16: abi.T2R_F16}


def _launch(dev, name, *args):
    """A C-ABI call on device index dev, its current stream as the last argument."""
    if dev == torch._C._cuda_getDevice():
        abi.call(name, *args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            abi.call(name, *args, torch._C._cuda_getCurrentRawStream(dev))


def _same(t, dev, dtype, what):
    if t.dtype is not dtype or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{what}: a contiguous {dtype} tensor on the rows' device")


def _rows(x, n, what):
    """(elements from row to row, dtype code, device index) of rows x [rows, n] that may lie apart."""
    code = _DTYPES.get(x.dtype)
    if code is None or x.dim() != 2 or x.shape[1] != n or not x.is_cuda:
        raise ValueError(f"{what}: float32, bfloat16 or float16 rows [rows, {n}] on a HIP device, not {x.dtype} {tuple(x.shape)}")
    ld, one = x.stride()
    if one != 1 and n > 1:
        raise ValueError(f"{what}: the values of a row lie side by side (stride 1, not {one})")
    return (ld if x.shape[0] > 1 else n), code, x.get_device()


_CACHE = "cache: kc [blocks, Hk, block, hd] and vc [blocks, Hk, hd, block] int8, ks and vs [blocks, Hk] float32, table [B, width] int32"


def _cache(dev, kc, vc, ks, vs, table):
    """The cache's arguments of the C-ABI and the table's sequences, after a check of its tensors."""
    if kc.dim() != 4 or table.dim() != 2:
        raise ValueError(_CACHE)
    n, Hk, block, hd = kc.shape
    B, width = table.shape
    if vc.shape != (n, Hk, hd, block) or ks.shape != (n, Hk) or vs.shape != ks.shape:
        raise ValueError(_CACHE)
    if kc.dtype is not I8 or vc.dtype is not I8 or ks.dtype is not F32 or vs.dtype is not F32 or table.dtype is not I32:
        raise ValueError(_CACHE)
    if not (kc.get_device() == vc.get_device() == ks.get_device() == vs.get_device() == table.get_device() == dev):
        raise ValueError("cache and table: on the rows' device")
    if not (kc.is_contiguous() and vc.is_contiguous() and ks.is_contiguous() and vs.is_contiguous() and table.is_contiguous()):
        raise ValueError("cache and table: contiguous tensors")
    return (kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr(), n, block, Hk, hd, table.data_ptr(), width), B


@functools.lru_cache(maxsize=1024)
def _workspace(name, *sizes):
    """Bytes of workspace that a call of these sizes needs (0 where it refuses them: the call itself then says so)."""
    return max(getattr(abi.load(), name)(*sizes), 0)


def _ragged(dev, B, starts, lens):
    _same(starts, dev, I32, "starts")
    _same(lens, dev, I32, "lens")
    if starts.dim() != 1 or lens.dim() != 1 or starts.numel() != B + 1 or lens.numel() != B:
        raise ValueError(f"starts [{B + 1}] and lens [{B}] for a table of {B} sequences")


def block_cache(n_blocks, Hk, hd, block=64, device="cuda:0"):
    """An empty block-scaled KV cache of n_blocks blocks of `block` tokens (16, 32, 64 or 128), Hk KV heads of hd (a
    multiple of 16, at most 128): kc [n_blocks, Hk, block, hd] and vc [n_blocks, Hk, hd, block] int8, ks and vs
    [n_blocks, Hk] float32. Which block holds which tokens is the caller's table [B, width] int32: position p of sequence
    b lies in block table[b, p // block], slot p % block; an entry outside the pool (-1) is no block."""
    z = lambda dt, *shape: torch.zeros(shape, dtype=dt, device=device)
    return z(I8, n_blocks, Hk, block, hd), z(I8, n_blocks, Hk, hd, block), z(F32, n_blocks, Hk), z(F32, n_blocks, Hk)


def kv_append_block(k, v, kc, vc, ks, vs, table, starts, lens):
    """Rows k, v [rows, Hk * hd] into the cache (t2r_kv_append_blk): those of sequence b are starts[b] .. starts[b + 1] - 1
    and the last of them gets position lens[b] - 1 (lens counts them). A block's scale for a head is max |x| / 127 over what
    it holds; it grows with later rows, and the block's earlier codes then move to it. Rows at places that the table has
    no block for are dropped. A block that rows enter stands in one place of one sequence: what two sequences share are full
    blocks, and a copy of the last one is the caller's."""
    n = kc.shape[1] * kc.shape[3] if kc.dim() == 4 else 0
    k_ld, code, dev = _rows(k, n, "k")
    v_ld, vcode, vdev = _rows(v, n, "v")
    if vcode != code or vdev != dev or v.shape != k.shape:
        raise ValueError("k and v: rows of one type, shape and device")
    cache, B = _cache(dev, kc, vc, ks, vs, table)
    _ragged(dev, B, starts, lens)
    if k.shape[0] and B:
        _launch(dev, "t2r_kv_append_blk", k.data_ptr(), v.data_ptr(), code, k_ld, v_ld, *cache, starts.data_ptr(),
                lens.data_ptr(), B, k.shape[0])


def kv_read_block(kc, vc, ks, vs, table, starts, lens, rows, dtype=torch.float32):
    """The cached values as rows k, v [rows, Hk * hd] (t2r_kv_read_blk): rows starts[b] .. starts[b + 1] - 1 are the last
    positions of sequence b, up to lens[b] - 1; zeros at places that the table has no block for. rows = starts[-1]; rows
    past it are not written."""
    if dtype not in _DTYPES:
        raise ValueError(f"kv_read_block gives float32, bfloat16 or float16, not {dtype}")
    if not kc.is_cuda:
        raise ValueError("op arguments must be contiguous tensors on a HIP device")
    dev = kc.get_device()
    cache, B = _cache(dev, kc, vc, ks, vs, table)
    _ragged(dev, B, starts, lens)
    k = torch.empty(rows, kc.shape[1] * kc.shape[3], dtype=dtype, device=kc.device)
    v = torch.empty_like(k)
    if rows and B:
        _launch(dev, "t2r_kv_read_blk", *cache, starts.data_ptr(), lens.data_ptr(), B, int(rows), _DTYPES[dtype],
                k.data_ptr(), v.data_ptr())
    return k, v


def _attention_block(q, cache, starts, lens, H, scale):
    hd = cache[0].shape[3] if cache[0].dim() == 4 else 0
    q_ld, code, dev = _rows(q, H * hd, "q")
    c, B = _cache(dev, *cache)
    rows = q.shape[0]
    if starts is not None:
        _ragged(dev, B, starts, lens)
    else:
        _same(lens, dev, I32, "lens")
        if lens.dim() != 1 or lens.numel() != B or rows != B:
            raise ValueError(f"one row of q and one length for each of the table's {B} sequences")
    where = q.device
    out = torch.empty(rows, H * hd, dtype=q.dtype, device=where)
    if not rows or not B:
        return out
    need = _workspace("t2r_attn_blk_workspace_bytes", B, 0 if starts is None else rows, H, c[6], hd, c[5], c[9], code)
    ws = torch.empty(need, dtype=torch.uint8, device=where) if need else None
    tail = (H, 1 / math.sqrt(hd) if scale is None else float(scale), out.data_ptr(), H * hd, ws.data_ptr() if need else None, need)
    if starts is None:
        _launch(dev, "t2r_attn_blk_decode", q.data_ptr(), code, q_ld, *c, lens.data_ptr(), B, *tail)
    else:
        _launch(dev, "t2r_attn_blk_prefill", q.data_ptr(), code, q_ld, *c, starts.data_ptr(), lens.data_ptr(), B, rows, *tail)
    return out


def attention_block(q, kc, vc, ks, vs, table, lens, H, scale=None):
    """Attention of one row a sequence, q [B, H * hd], over positions 0 .. lens[b] - 1 of the block-scaled cache
    (t2r_attn_blk_decode): softmax(scale q K^T) V with scale 1 / sqrt(hd) unless given; H a multiple of Hk. A row whose
    sequence is empty gives zeros."""
    return _attention_block(q, (kc, vc, ks, vs, table), None, lens, H, scale)


def attention_block_prefill(q, kc, vc, ks, vs, table, starts, lens, H, scale=None):
    """Attention of ragged rows q [rows, H * hd] over the block-scaled cache (t2r_attn_blk_prefill): rows starts[b] ..
    starts[b + 1] - 1 are the last positions of sequence b, up to lens[b] - 1, already in the cache; each sees the positions
    up to its own. A row below position 0 (lens[b] less than the sequence's rows) gives NaN; rows past starts[-1] are not
    written."""
    return _attention_block(q, (kc, vc, ks, vs, table), starts, lens, H, scale)


# ------------------------------------------------------------------ log probabilities
def logprobs(logits, tokens=None, top=0):
    """Of logits rows [rows, V] (t2r_logprobs): (log softmax at tokens [rows] int32, or None without tokens; the entropy;
    the ids [rows, top] and the log probabilities of the `top` <= 32 largest, descending, the lower id first on ties), all
    float32 and int32. A token outside [0, V) gives NaN; logits of -inf have probability 0."""
    if logits.dim() != 2:
        raise ValueError("logits: rows [rows, V]")
    rows, V = logits.shape
    ld, code, dev = _rows(logits, V, "logits")
    where = logits.device
    lp = None
    if tokens is not None:
        _same(tokens, dev, I32, "tokens")
        if tokens.dim() != 1 or tokens.numel() != rows:
            raise ValueError(f"one token for each of the {rows} rows")
        lp = torch.empty(rows, dtype=F32, device=where)
    if not 0 <= top <= min(V, 32):
        raise ValueError(f"top {top}: 0 .. {min(V, 32)} of {V} values")
    ent = torch.empty(rows, dtype=F32, device=where)
    ids = torch.empty(rows, top, dtype=I32, device=where)
    val = torch.empty(rows, top, dtype=F32, device=where)
    if rows:
        need = _workspace("t2r_logprobs_workspace_bytes", rows, V, top)
        ws = torch.empty(need, dtype=torch.uint8, device=where) if need else None
        _launch(dev, "t2r_logprobs", logits.data_ptr(), code, ld, abi.ptr(tokens), rows, V, top, abi.ptr(lp), ent.data_ptr(),
                ids.data_ptr(), val.data_ptr(), ws.data_ptr() if need else None, need)
    return lp, ent, ids, val
