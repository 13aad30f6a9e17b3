"""Refusals and host-side arithmetic of the paged-KV operators (no GPU needed)."""
import ctypes
import math

import pytest
import torch

from unified_cache_management_b200 import lib as L
from unified_cache_management_b200 import ops

NULL = None
P = 0x1000          # an aligned address that is never read: every call below is refused before a launch


def _rotary(lib, **kw):
    a = dict(x=P, out=P, T=4, H=2, D=64, xt=128, xh=64, ot=128, oh=64, dtype=L.BF16, pos=P, p64=1, f=P, rot=64, inter=0, m=1.0, tr=0)
    a.update(kw)
    return lib.ucmr_rotary(*a.values(), NULL)


def test_rotary_refusals():
    lib = L.load_library()
    for kw in (dict(x=NULL), dict(out=NULL), dict(pos=NULL), dict(f=NULL), dict(T=-1), dict(D=0), dict(rot=0), dict(rot=3), dict(rot=66)):
        assert _rotary(lib, **kw) == L.UCMR_ERR_BAD_ARG, kw
    assert _rotary(lib, dtype=L.E4M3) == L.UCMR_ERR_UNSUPPORTED
    assert _rotary(lib, T=0, x=NULL) == L.UCMR_OK


def _append(lib, **kw):
    a = dict(k=P, kt=128, kh=64, v=P, vt=128, vh=64, T=4, H=2, D=64, dtype=L.BF16, slots=P, s64=1, kc=P, kcb=2048, kct=128, kch=64,
             vc=P, vcb=2048, vct=128, vch=64, NB=8, BS=16, cache=L.E4M3, ks=P, vs=P, pos=P, p64=1, f=P, rot=64, inter=0, m=1.0, q=NULL,
             hq=0, qt=0, qh=0, qo=NULL, qot=0, qoh=0, ko=NULL, kot=0, koh=0)
    a.update(kw)
    return lib.ucmr_kv_append(*a.values(), NULL)


def test_append_refusals():
    lib = L.load_library()
    for kw in (dict(k=NULL), dict(v=NULL), dict(slots=NULL), dict(kc=NULL), dict(vc=NULL), dict(ks=NULL), dict(vs=NULL), dict(pos=NULL),
               dict(T=-1), dict(H=0), dict(BS=0), dict(NB=-1), dict(rot=0), dict(rot=80), dict(f=NULL, q=P, hq=2, qo=P), dict(f=NULL, ko=P),
               dict(q=P, hq=2), dict(q=P, hq=0, qo=P), dict(ko=P), dict(cache=L.BF16)):
        assert _append(lib, **kw) == L.UCMR_ERR_BAD_ARG, kw
    for kw in (dict(dtype=L.E4M3), dict(cache=L.FP16, ks=NULL, vs=NULL), dict(D=72, rot=64), dict(D=1024), dict(BS=2048), dict(rot=24),
               dict(k=P + 2), dict(kt=132), dict(kct=136), dict(vcb=2056), dict(v=P + 8)):
        assert _append(lib, **kw) == L.UCMR_ERR_UNSUPPORTED, kw
    assert _append(lib, T=0, k=NULL) == L.UCMR_OK


def _attention(lib, **kw):
    a = dict(q=P, T=3, Hq=4, D=128, qt=512, qh=128, dtype=L.BF16, kc=P, kcb=4096, kct=256, kch=128, vc=P, vcb=4096, vct=256, vch=128,
             NB=9, BS=16, Hkv=2, cache=L.E4M3, ks=P, vs=P, table=P, mb=4, btb=4, bth=0, lens=P, start=NULL, mq=1, B=3, scale=0.1, causal=1,
             out=P, ot=512, oh=128, lse=NULL, ws=P, wsb=1 << 30)
    a.update(kw)
    return lib.ucmr_paged_attention(*a.values(), NULL)


def test_attention_refusals():
    lib = L.load_library()
    for kw in (dict(q=NULL), dict(kc=NULL), dict(vc=NULL), dict(table=NULL), dict(lens=NULL), dict(out=NULL), dict(ks=NULL), dict(vs=NULL),
               dict(T=4), dict(Hq=5), dict(Hkv=0), dict(D=0), dict(BS=0), dict(B=-1), dict(mb=-1), dict(cache=L.BF16)):
        assert _attention(lib, **kw) == L.UCMR_ERR_BAD_ARG, kw
    for kw in (dict(D=96), dict(dtype=L.E4M3), dict(cache=L.FP16, ks=NULL, vs=NULL), dict(kc=P + 8), dict(kct=264), dict(q=P + 2), dict(oh=132),
               dict(mb=1 << 30)):
        assert _attention(lib, **kw) == L.UCMR_ERR_UNSUPPORTED, kw
    for kw in (dict(ws=NULL), dict(wsb=4096)):
        assert _attention(lib, **kw) == L.UCMR_ERR_WORKSPACE, kw
    assert _attention(lib, T=0, B=0, q=NULL) == L.UCMR_OK
    need = lib.ucmr_paged_attention_workspace_bytes(128)
    assert need > lib.ucmr_paged_attention_workspace_bytes(64) > L.WORKSPACE_HEADER_BYTES
    assert lib.ucmr_paged_attention_workspace_bytes(0) == 0
    assert lib.ucmr_paged_attention_workspace_init(NULL, need, NULL) == L.UCMR_ERR_WORKSPACE
    assert lib.ucmr_paged_attention_workspace_init(ctypes.c_void_p(P), 64, NULL) == L.UCMR_ERR_WORKSPACE


def test_wrappers_want_cuda_tensors():
    x, i = torch.zeros((2, 2, 64), dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int64)
    f, _ = ops.rotary_frequencies(64)
    c = torch.zeros((3, 16, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ops.rotary(x, i, f)
    with pytest.raises(ValueError):
        ops.kv_append(x, x, i, c, c)
    with pytest.raises(ValueError):
        ops.paged_attention(x, c, c, torch.zeros((2, 3), dtype=torch.int32), torch.zeros(2, dtype=torch.int32))


def test_rotary_frequencies():
    f, m = ops.rotary_frequencies(128, 10000.0)
    assert m == 1.0 and f.dtype == torch.float64 and f[0] == 1.0
    assert torch.allclose(f[1:] / f[:-1], torch.full((63,), 10000.0 ** (-1 / 64), dtype=torch.float64), rtol=1e-13)
    lin, _ = ops.rotary_frequencies(128, 10000.0, {"type": "linear", "factor": 4.0})
    assert torch.allclose(lin, f / 4, rtol=1e-15)
    # dynamic: unchanged inside the original context; beyond it the slowest pair is stretched by factor*ratio - (factor - 1)
    dyn = {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 4096}
    assert torch.equal(ops.rotary_frequencies(128, 10000.0, dict(dyn, seq_len=1000))[0], f)
    far, _ = ops.rotary_frequencies(128, 10000.0, dict(dyn, seq_len=16384))
    assert math.isclose(float(f[-1] / far[-1]), 2.0 * 4 - 1, rel_tol=1e-12) and far[0] == 1.0
    # llama3: fast pairs keep their frequency, slow ones are divided by the factor, monotone between
    l3, m = ops.rotary_frequencies(128, 500000.0, {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0,
                                                   "high_freq_factor": 4.0, "original_max_position_embeddings": 8192})
    g, _ = ops.rotary_frequencies(128, 500000.0)
    wave = 2 * math.pi / g
    assert m == 1.0 and torch.equal(l3[wave < 8192 / 4], g[wave < 8192 / 4])
    assert torch.allclose(l3[wave > 8192], g[wave > 8192] / 8, rtol=1e-15) and (l3[1:] < l3[:-1]).all()
    # yarn: ramp between the pairs of 32 turns and 1 turn, and the factor on the values
    y, m = ops.rotary_frequencies(128, 10000.0, {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096})
    assert math.isclose(m, 0.1 * math.log(40.0) + 1.0) and torch.equal(y[:20], f[:20]) and torch.allclose(y[46:], f[46:] / 40, rtol=1e-15)
    assert ops.rotary_frequencies(128, 10000.0, {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096,
                                                 "attention_factor": 1.0})[1] == 1.0
    for bad in (dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=8, scaling={"type": "odd"}), dict(rotary_dim=8, scaling={"type": "linear", "factor": 0})):
        with pytest.raises(ValueError):
            ops.rotary_frequencies(**bad)


def test_yarn_entries():
    """Every key of a yarn entry counts: the factor from mscale and mscale_all_dim, ends of the ramp that are not rounded."""
    yarn = {"type": "yarn", "factor": 40, "original_max_position_embeddings": 4096, "beta_fast": 32, "beta_slow": 1}
    plain, m = ops.rotary_frequencies(64, 10000.0, yarn)
    assert math.isclose(m, 0.1 * math.log(40.0) + 1.0)

    def s(x):
        return 0.1 * x * math.log(40.0) + 1.0
    for one, every in ((0.707, 0.707), (1.0, 1.0), (1.0, 0.5), (0.707, 2.0)):
        f, m = ops.rotary_frequencies(64, 10000.0, dict(yarn, mscale=one, mscale_all_dim=every))
        assert math.isclose(m, s(one) / s(every), rel_tol=1e-14) and torch.equal(f, plain)
    assert ops.rotary_frequencies(64, 10000.0, dict(yarn, mscale=0.707, mscale_all_dim=1.0, attention_factor=1.5))[1] == 1.5
    assert ops.rotary_frequencies(64, 10000.0, dict(yarn, factor=1.0, mscale=0.707, mscale_all_dim=1.0))[1] == 1.0
    assert math.isclose(ops.rotary_frequencies(64, 10000.0, dict(yarn, mscale=1.0, mscale_all_dim=0.0))[1], s(1.0))
    # the ramp runs from the pair of 32 turns to that of 1 turn over the original context: fractional unless truncated
    f = 10000.0 ** (-2.0 * torch.arange(32, dtype=torch.float64) / 64)
    lo, hi = (64 * math.log(4096 / (2 * math.pi * t)) / (2 * math.log(10000.0)) for t in (32.0, 1.0))
    for cut in (True, False):
        a, b = (math.floor(lo), math.ceil(hi)) if cut else (lo, hi)
        slow = ((torch.arange(32, dtype=torch.float64) - a) / (b - a)).clamp(0, 1)
        got, _ = ops.rotary_frequencies(64, 10000.0, dict(yarn, truncate=cut))
        assert torch.allclose(got, f * (1 - slow) + f / 40 * slow, rtol=1e-14)
    assert not torch.equal(ops.rotary_frequencies(64, 10000.0, dict(yarn, truncate=False))[0], plain)
    # keys without a value are not there; what is not handled, contradicts the base or is defined in two ways is refused
    assert torch.equal(ops.rotary_frequencies(64, 10000.0, dict(yarn, attention_factor=None, mrope_section=None, rope_theta=10000))[0], plain)
    for bad in (dict(mscale=0.707), dict(mscale_all_dim=1.0), dict(mscale=0.707, mscale_all_dim=0.0), dict(rope_theta=5e5),
                dict(mrope_section=[16, 24, 24]), dict(alpha=2.0)):
        with pytest.raises(ValueError):
            ops.rotary_frequencies(64, 10000.0, dict(yarn, **bad))
    with pytest.raises(ValueError):
        ops.rotary_frequencies(64, 10000.0, {"rope_type": "default", "mrope_section": [16, 24, 24]})


def test_append_token_limit():
    """The walk of the slot list grows with the square of the tokens: a call has a limit."""
    lib = L.load_library()
    for cache in (dict(), dict(cache=L.BF16, ks=NULL, vs=NULL)):
        assert _append(lib, T=(1 << 22) + 1, **cache) == L.UCMR_ERR_UNSUPPORTED
        assert _append(lib, T=1 << 40, **cache) == L.UCMR_ERR_UNSUPPORTED
