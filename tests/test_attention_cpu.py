"""Argument checks of the attention and 8-bit cache entry points that need no GPU: the C calls refuse before anything is launched, the Python ones
before the library is reached."""
import ctypes

import pytest
import torch


def _args(**kw):
    from aesrc2020_amd.attention import Xattn
    a = Xattn()
    base = dict(q=4096, k=4096, v=4096, out=4096, B=2, Tq=3, Tk=70, Hq=4, Hkv=2, D=64, scale=0.125, q_sb=768, q_st=256, q_sh=64, k_sb=8960, k_st=128, k_sh=64,
                v_sb=8960, v_st=128, v_sh=64, o_sb=768, o_st=256, o_sh=64)
    for n, v in {**base, **kw}.items():
        setattr(a, n, v)
    return a


BAD = [dict(D=12), dict(D=136), dict(D=0), dict(B=0), dict(Tq=0), dict(Tk=-1), dict(Hq=3), dict(Hkv=0), dict(q=None), dict(out=None), dict(q=4104), dict(k=4100), dict(q_st=257),
       dict(v_sh=-64), dict(Tq=1 << 30), dict(B=1 << 24, Tq=100)]


@pytest.mark.parametrize("sfx", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kw", BAD, ids=lambda k: "-".join("%s=%s" % i for i in k.items()))
def test_c_forward_and_backward_refuse(sfx, kw):
    from aesrc2020_amd import _lib
    L = _lib.lib().fn
    a = _args(**kw)
    assert L["sar_xattn_fwd_" + sfx](ctypes.byref(a), None) == -1
    for n in ("lse", "dout", "dq", "dk", "dv", "ws"):
        setattr(a, n, 4096)
    a.ws_bytes = 1 << 40
    assert L["sar_xattn_bwd_" + sfx](ctypes.byref(a), None) == -1


@pytest.mark.parametrize("sfx", ["f32", "bf16", "f16"])
def test_c_refuses_missing_and_small_workspaces(sfx):
    from aesrc2020_amd import _lib
    L = _lib.lib().fn
    a = _args(B=1, Tk=5000, Tq=1)                                  # few rows, many keys: the key axis is cut
    need = L["sar_xattn_fwd_workspace_bytes"](ctypes.byref(a))
    assert need > 0
    for ws, n in ((None, 0), (4096, need - 1), (4104, need), (4096, -1)):
        a.ws, a.ws_bytes = ws, n
        assert L["sar_xattn_fwd_" + sfx](ctypes.byref(a), None) == -1
    a = _args(lse=4096, dout=4096, dq=4096, dk=4096, dv=4096, ws=4096)
    need = L["sar_xattn_bwd_workspace_bytes"](ctypes.byref(a))
    a.ws_bytes = need - 1
    assert need > 0 and L["sar_xattn_bwd_" + sfx](ctypes.byref(a), None) == -1
    a.ws_bytes, a.lse = need, None
    assert L["sar_xattn_bwd_" + sfx](ctypes.byref(a), None) == -1
    assert L["sar_xattn_fwd_workspace_bytes"](ctypes.byref(_args(D=7))) == 0


def test_c_workspace_sizes():
    """No keys, one key, the largest calls: sizes that hold every slice and overflow nothing."""
    from aesrc2020_amd import _lib
    L = _lib.lib().fn
    size = lambda **kw: L["sar_xattn_bwd_workspace_bytes"](ctypes.byref(_args(**kw)))  # noqa: E731
    assert size(Tk=0) == 256 and size(Tk=1) == 256                 # {lse, delta} of 2 x 4 x 3 rows
    assert size(B=1, Tq=1000, Tk=0) == 8 * 4000
    assert size(B=1, Tq=100, Tk=4000, Hq=2) > 8 * 200 + 4 * 100 * 2 * 64                   # dQ in slices
    for kw in (dict(B=1, Tq=1, Tk=t, D=d) for t in (256, 257, 700, 1100, 1700, 5000) for d in (32, 64, 128)):
        for q in ("sar_xattn_fwd_workspace_bytes", "sar_kv8_attend_workspace_bytes"):
            most, two, four = (L[q](ctypes.byref(_args(elt_bytes=e, **kw))) for e in (0, 2, 4))
            assert two <= four == most and (kw["Tk"] > 256 or most == 0), (kw, q)
    assert size(B=1024, Hq=32, Hkv=32, Tq=4096, Tk=4096, D=128) == 8 * 1024 * 32 * 4096


@pytest.mark.parametrize("sfx", ["f32", "bf16", "f16"])
def test_c_cache_refuses(sfx):
    from aesrc2020_amd import _lib
    L = _lib.lib().fn
    store = lambda k=4096, st=128, k8=4096, T=64, D=64, frames=128, first=0, lens_out=4096: L["sar_kv8_store_" + sfx](  # noqa: E731
        k, 8192, st, 64, 4096, 8192, 128, 64, None, k8, 4096, 4096, 4096, lens_out, 2, T, 2, D, frames, first, None)
    for kw in (dict(k=None), dict(k=4097), dict(st=129), dict(k8=None), dict(T=0), dict(D=20), dict(frames=100), dict(first=32), dict(first=128), dict(T=129), dict(lens_out=None)):
        assert store(**kw) == -1, kw
    at = lambda a, frames=128, k8=4096: L["sar_kv8_attend_" + sfx](ctypes.byref(a), k8, 4096, 4096, 4096, frames, None)  # noqa: E731
    assert at(_args(), frames=64) == -1 and at(_args(), frames=100) == -1 and at(_args(), k8=None) == -1 and at(_args(q=4098)) == -1 and at(_args(q_st=3)) == -1 and at(_args(D=4)) == -1
    assert at(_args(B=1, Tk=5000), frames=5056) == -1              # no workspace given


def test_python_refuses_what_is_not_on_a_device():
    from aesrc2020_amd import attention as A
    q, k = torch.zeros(1, 2, 2, 16), torch.zeros(1, 3, 2, 16)
    with pytest.raises(ValueError, match="no CPU fallback"):
        A.cross_attention(q, k, k)
    with pytest.raises(ValueError, match="batch, time, heads"):
        A.cross_attention(q[0], k, k)
    with pytest.raises(ValueError, match="float32"):
        A.cross_attention(q.double(), k, k)
    with pytest.raises(ValueError, match="multiple of 8"):
        A.EncoderCache8(1, 10, 2, 20, device="cpu")
