"""Argument checks of the vocabulary cross entropy that need no GPU: refused before anything is launched."""
import ctypes

import pytest
import torch


def _args(**kw):
    from aesrc2020_amd.losses import _VocabCe
    a = _VocabCe()
    for n, v in {**dict(x=4096, kernel=4096, labels=4096, dloss=4096, loss=4096, lse=4096, dx=4096, dkernel=4096, ws=4096, ws_bytes=1 << 40, ldx=64, ldk=1000, R=10, D=64, V=1000,
                        label_bytes=4), **kw}.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("sfx", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kw", [dict(x=None), dict(kernel=None), dict(labels=None), dict(R=0), dict(D=0), dict(V=0), dict(ldx=63), dict(ldk=999), dict(label_bytes=2), dict(ws=None),
                                dict(ws=4100), dict(ws_bytes=100), dict(R=1 << 25), dict(V=1 << 25, ldk=1 << 25), dict(ldx=1 << 23), dict(R=1 << 22, V=1 << 22, ldk=1 << 22)], ids=lambda k: "-".join("%s=%s" % i for i in k.items()))
def test_c_refuses(sfx, kw):
    from aesrc2020_amd import _lib
    L = _lib.lib().fn
    a = _args(**kw)
    assert L["sar_vocab_ce_fwd_" + sfx](ctypes.byref(a), None) == -1 and L["sar_vocab_ce_bwd_" + sfx](ctypes.byref(a), None) == -1


@pytest.mark.parametrize("sfx", ["f32", "bf16", "f16"])
def test_c_refuses_by_direction_and_bounds_the_workspace(sfx):
    from aesrc2020_amd import _lib
    L = _lib.lib().fn
    assert L["sar_vocab_ce_fwd_" + sfx](ctypes.byref(_args(loss=None, lse=None)), None) == -1
    for kw in (dict(lse=None), dict(dloss=None), dict(dx=None, dkernel=None)):
        assert L["sar_vocab_ce_bwd_" + sfx](ctypes.byref(_args(**kw)), None) == -1
    if sfx != "f32":
        assert L["sar_vocab_ce_bwd_" + sfx](ctypes.byref(_args(accumulate=1)), None) == -1
    # the logits of 65536 rows over 200000 classes would be 52 GB in fp32: the call's workspace stays a small part of that
    big = _args(R=65536, D=256, V=200000, ldx=256, ldk=200000)
    assert 0 < L["sar_vocab_ce_bwd_%s_workspace_bytes" % sfx](ctypes.byref(big)) < 2 << 30
    assert L["sar_vocab_ce_fwd_%s_workspace_bytes" % sfx](ctypes.byref(_args(V=0))) == 0


def test_python_refuses_what_is_not_on_a_device():
    from aesrc2020_amd.losses import vocab_crossentropy
    with pytest.raises(ValueError, match="HIP device"):
        vocab_crossentropy(torch.zeros(2, 8), torch.zeros(8, 5), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="vocabulary"):
        vocab_crossentropy(torch.zeros(2, 8), torch.zeros(9, 5), torch.zeros(2, dtype=torch.int32))
