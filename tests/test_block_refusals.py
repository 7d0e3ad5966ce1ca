"""What the block-cache and log-probability calls refuse, before anything is launched (no GPU needed), and that the float64
restatement which their GPU tests compare with does what the definitions say."""
import ctypes

import numpy as np
import pytest

import blockref
from t2r_amd import abi

P = ctypes.c_void_p(4096)
ODD = ctypes.c_void_p(4098)


def append(lib, **kw):
    a = dict(k=P, v=P, dtype=0, k_ld=128, v_ld=128, kc=P, vc=P, ks=P, vs=P, n=4, block=64, Hk=2, hd=64, table=P, width=2, starts=P,
             lens=P, B=1, rows=1)
    a.update(kw)
    return lib.t2r_kv_append_blk(*a.values(), None)


def attend(lib, form, **kw):
    a = dict(q=P, dtype=0, q_ld=256, kc=P, vc=P, ks=P, vs=P, n=4, block=64, Hk=2, hd=64, table=P, width=2)
    a.update(starts=P) if form == "prefill" else None
    a.update(lens=P, B=1)
    a.update(rows=1) if form == "prefill" else None
    a.update(H=4, scale=0.125, out=P, out_ld=256, ws=None, ws_bytes=0)
    a.update(kw)
    return getattr(lib, "t2r_attn_blk_" + form)(*a.values(), None)


BAD_CACHE = [(dict(kc=None), abi.T2R_EINVAL), (dict(vs=None), abi.T2R_EINVAL), (dict(table=None), abi.T2R_EINVAL),
             (dict(lens=None), abi.T2R_EINVAL), (dict(kc=ctypes.c_void_p(4104)), abi.T2R_EINVAL), (dict(dtype=3), abi.T2R_EINVAL),
             (dict(block=48), abi.T2R_ESHAPE), (dict(block=256), abi.T2R_ESHAPE), (dict(block=0), abi.T2R_ESHAPE),
             (dict(hd=72), abi.T2R_ESHAPE), (dict(hd=144), abi.T2R_ESHAPE), (dict(hd=0), abi.T2R_ESHAPE),
             (dict(Hk=0), abi.T2R_ESHAPE), (dict(n=0), abi.T2R_ESHAPE), (dict(width=0), abi.T2R_ESHAPE),
             (dict(n=1 << 30, Hk=4), abi.T2R_ESHAPE), (dict(width=1 << 26), abi.T2R_ESHAPE), (dict(B=0), abi.T2R_ESHAPE)]


@pytest.mark.parametrize("kw,code", BAD_CACHE + [(dict(rows=0), abi.T2R_ESHAPE), (dict(rows=1 << 24), abi.T2R_ESHAPE),
                                                 (dict(k_ld=127), abi.T2R_ESHAPE), (dict(v_ld=64), abi.T2R_ESHAPE), (dict(v=ODD), abi.T2R_EINVAL),
                                                 (dict(starts=None), abi.T2R_EINVAL)])
def test_append_refuses(kw, code):
    assert append(abi.load(), **kw) == code


@pytest.mark.parametrize("form", ["decode", "prefill"])
@pytest.mark.parametrize("kw,code", BAD_CACHE + [(dict(H=5), abi.T2R_ESHAPE), (dict(H=66), abi.T2R_ESHAPE), (dict(H=0), abi.T2R_ESHAPE),
                                                 (dict(scale=0.0), abi.T2R_EINVAL), (dict(scale=-1.0), abi.T2R_EINVAL),
                                                 (dict(scale=float("nan")), abi.T2R_EINVAL), (dict(scale=float("inf")), abi.T2R_EINVAL),
                                                 (dict(q_ld=255), abi.T2R_ESHAPE), (dict(out_ld=255), abi.T2R_ESHAPE),
                                                 (dict(out=None), abi.T2R_EINVAL), (dict(q=ODD), abi.T2R_EINVAL),
                                                 (dict(width=64), abi.T2R_ENOMEM), (dict(width=64, ws=P, ws_bytes=100), abi.T2R_ENOMEM),
                                                 (dict(width=64, ws=ctypes.c_void_p(4100), ws_bytes=1 << 30), abi.T2R_ENOMEM)])
def test_attention_refuses(form, kw, code):
    assert attend(abi.load(), form, **kw) == code


def test_attention_refuses_its_own():
    lib = abi.load()
    assert attend(lib, "decode", B=65536) == abi.T2R_ESHAPE
    assert attend(lib, "decode", width=1 << 20) == abi.T2R_ENOMEM and attend(lib, "decode", width=1 << 22) == abi.T2R_ESHAPE
    assert attend(lib, "prefill", rows=0) == abi.T2R_ESHAPE and attend(lib, "prefill", rows=1 << 24) == abi.T2R_ESHAPE
    # (more workgroups than a launch has threads for: 2^23 rows in tiles of one row and 4 KV heads)
    assert attend(lib, "prefill", rows=1 << 23, H=128, Hk=4, hd=128, q_ld=1 << 14, out_ld=1 << 14, width=64) == abi.T2R_ESHAPE
    assert attend(lib, "prefill", starts=None) == abi.T2R_EINVAL
    assert lib.t2r_attn_blk_workspace_bytes(1, 0, 4, 2, 64, 64, 2, 0) == 0
    assert lib.t2r_attn_blk_workspace_bytes(1, 0, 4, 2, 64, 64, 128, 0) > 0
    assert lib.t2r_attn_blk_workspace_bytes(0, 0, 4, 2, 64, 64, 128, 0) == -1
    assert lib.t2r_attn_blk_workspace_bytes(1, 0, 5, 2, 64, 64, 128, 0) == -1


@pytest.mark.parametrize("form", ["decode", "prefill"])
def test_attention_refuses_scales_past_the_kernels_range(form):
    """The kernels take scale log2(e): an infinity there would give NaN where q or a key is zero."""
    for scale, code in ((2.9e38, abi.T2R_EINVAL), (2.3e38, abi.T2R_ENOMEM)):       # (a second refusal follows: no workspace)
        assert attend(abi.load(), form, scale=scale, width=64) == code


@pytest.mark.parametrize("sizes", [
    (384, 384, 1, 1, 64, 1 << 30, 1 << 30, 0),                             # (a cut of 2^32 keys is 0 in 32 bits)
    (1, 0, 4, 2, 64, 48, 100, 0), (1, 0, 4, 2, 72, 64, 100, 0), (1, 0, 4, 2, 144, 64, 100, 0), (1, 0, 4, 2, 64, 128, 1 << 24, 0),
    (1, 0, 4, 2, 64, 64, 1 << 22, 0), (65536, 0, 4, 2, 64, 64, 100, 0), (1, 0, 1 << 17, 1 << 16, 64, 64, 100, 0),
    (1, 1 << 24, 4, 2, 64, 64, 100, 0), (1, -1, 4, 2, 64, 64, 100, 0), (1, 1 << 23, 128, 4, 128, 64, 64, 0),
    (2 ** 31 - 1, 0, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1, 0), (1, 0, 4, 2, 64, 64, 100, 3)])
def test_attention_workspace_of_sizes_that_the_calls_refuse(sizes):
    assert abi.load().t2r_attn_blk_workspace_bytes(*sizes) == -1


@pytest.mark.parametrize("sizes", [(1000, 20000, 33), (1, 2 ** 31 - 1, 5), (1, 2, 3), (1 << 24, 100, 1), (1, 20000, -1),
                                   (2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1)])
def test_logprobs_workspace_of_sizes_that_the_call_refuses(sizes):
    assert abi.load().t2r_logprobs_workspace_bytes(*sizes) == -1


def test_read_refuses():
    lib = abi.load()
    ok = dict(kc=P, vc=P, ks=P, vs=P, n=4, block=64, Hk=2, hd=64, table=P, width=2, starts=P, lens=P, B=1, rows=1, dtype=0, k=P, v=P)
    for kw, code in BAD_CACHE + [(dict(rows=0), abi.T2R_ESHAPE), (dict(rows=1 << 24), abi.T2R_ESHAPE), (dict(k=None), abi.T2R_EINVAL)]:
        assert lib.t2r_kv_read_blk(*{**ok, **kw}.values(), None) == code


def test_logprobs_refuses():
    lib = abi.load()
    ok = dict(x=P, dtype=0, ld=100, tokens=P, rows=2, V=100, top=3, lp=P, ent=P, ids=P, val=P, ws=P, ws_bytes=1 << 20)
    for kw, code in ((dict(x=None), abi.T2R_EINVAL), (dict(tokens=None), abi.T2R_EINVAL), (dict(ids=None), abi.T2R_EINVAL),
                     (dict(val=None), abi.T2R_EINVAL), (dict(dtype=-1), abi.T2R_EINVAL), (dict(x=ODD), abi.T2R_EINVAL),
                     (dict(rows=0), abi.T2R_ESHAPE), (dict(rows=1 << 24), abi.T2R_ESHAPE), (dict(V=0), abi.T2R_ESHAPE), (dict(V=2 ** 31 - 1, ld=2 ** 31), abi.T2R_ESHAPE), (dict(ld=99), abi.T2R_ESHAPE),
                     (dict(top=-1), abi.T2R_ERANGE), (dict(top=33), abi.T2R_ERANGE), (dict(V=2, top=3), abi.T2R_ERANGE),
                     (dict(V=20000, ld=20000, ws=None), abi.T2R_ENOMEM), (dict(V=20000, ld=20000, ws_bytes=10), abi.T2R_ENOMEM)):
        assert lib.t2r_logprobs(*{**ok, **kw}.values(), None) == code, kw
    assert lib.t2r_logprobs_workspace_bytes(0, 5, 0) == -1 and lib.t2r_logprobs_workspace_bytes(1, 5, 0) == 0


def test_host_checks():
    """Tensors on the host, of other types, shapes or strides are refused by name."""
    import torch

    from t2r_amd import ops
    c = ops.block_cache(2, 2, 32, 16, device="cpu")
    x, table = torch.zeros((1, 64)), torch.zeros((1, 2), dtype=torch.int32)
    st, ln = torch.tensor([0, 1], dtype=torch.int32), torch.tensor([1], dtype=torch.int32)
    for call in (lambda: ops.kv_append_block(x, x, *c, table, st, ln), lambda: ops.attention_block(x, *c, table, ln, 2),
                 lambda: ops.attention_block_prefill(x, *c, table, st, ln, 2), lambda: ops.kv_read_block(*c, table, st, ln, 1),
                 lambda: ops.logprobs(x), lambda: ops.logprobs(x[0]), lambda: ops.kv_read_block(*c, table, st, ln, 1, dtype=torch.int8)):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------ the restatement itself
def test_reference_scale_follows_the_rows():
    c = blockref.Cache(2, 1, 16, 16)
    table = [[1, 0]]
    a = np.linspace(-1, 1, 16, dtype=np.float32)[None]
    c.append(a, 2 * a, table, [0, 1], [1])
    assert c.ks[1, 0] == np.float32(1 / 127) and c.vs[1, 0] == np.float32(2 / 127) and c.kc[1, 0, 0, 15] == 127
    c.append(4 * a, 0.5 * a, table, [0, 1], [2])
    assert c.ks[1, 0] == np.float32(4 / 127) and c.vs[1, 0] == np.float32(2 / 127)
    assert c.kc[1, 0, 0, 15] == 32 and c.kc[1, 0, 1, 15] == 127 and c.vc[1, 0, 15, 1] == 32      # 127 / 4 = 31.75
    k, v, there = c.values(table, 0, 2)
    assert there.all() and abs(k[1, 0, 15] - 4) < 1e-6 and abs(k[0, 0, 15] - 1) < 4 / 254 + 1e-6


def test_reference_attention_of_one_key_is_its_value():
    c = blockref.Cache(1, 1, 16, 16)
    x = np.arange(16, dtype=np.float32)[None]
    c.append(x, x, [[0]], [0, 1], [1])
    out, bound = blockref.attention(c, x, [[0]], [0, 1], [1], 1, 0.25)
    assert np.allclose(out, c.vc[0, 0, :, 0] * float(c.vs[0, 0])) and (bound >= 0).all()


def test_reference_logprobs_ties_and_bans():
    x = np.asarray([[1.0, 3.0, 3.0, -np.inf], [-np.inf] * 4])
    lp, ent, ids, val = blockref.logprobs(x, [2, 0], 3)
    assert ids[0].tolist() == [1, 2, 0] and ids[1].tolist() == [0, 1, 2]
    p = np.exp([1.0, 3.0, 3.0]) / np.exp([1.0, 3.0, 3.0]).sum()
    assert np.isclose(lp[0], np.log(p[2])) and np.isclose(ent[0], -(p * np.log(p)).sum()) and lp[1] == -np.inf and ent[1] == 0
