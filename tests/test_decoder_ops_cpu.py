"""Argument checks of the decoder operators that need no GPU."""
import ctypes

import pytest
import torch


def test_a_vector_that_has_to_be_given_is_not_made_up():
    from aesrc2020_amd.attention import _given
    t = torch.zeros(8)
    assert _given("lse", t[1:], (7,), torch.float32, t.device).data_ptr() == t.data_ptr() + 4        # a view on 4-byte boundaries will do
    for bad in (None, t, t[::2], t.double()[1:], t.view(7 + 1, 1)[1:]):
        with pytest.raises(ValueError, match="lse"):
            _given("lse", bad, (7,), torch.float32, t.device)


def test_missing_tensors_are_refused():
    from aesrc2020_amd.attention import cross_attention, cross_attention_grad
    from aesrc2020_amd.losses import vocab_crossentropy
    for f in (lambda: cross_attention(None, None, None), lambda: cross_attention_grad(None, None, None, None, None, None), lambda: vocab_crossentropy(None, None, None),
              lambda: vocab_crossentropy(torch.zeros(2, 8), torch.zeros(8, 5), None)):
        with pytest.raises(ValueError):
            f()


@pytest.mark.parametrize("sfx", ["f32", "bf16", "f16"])
def test_grids_of_more_threads_than_a_launch_takes_are_refused(sfx):
    """2^32 threads: 2^23 row tiles of 512 (few rows), 2^24 blocks of 256 (the gradients' rows, their keys)."""
    from aesrc2020_amd import _lib
    from tests.test_attention_cpu import _args
    L = _lib.lib().fn
    for kw in (dict(B=1 << 22, Tq=1, Hq=2, Hkv=2), dict(B=1 << 23, Tq=40, Hq=1, Hkv=1), dict(B=1 << 20, Tq=1, Tk=2048, Hq=1, Hkv=1)):
        a = _args(**kw)
        for n in ("lse", "dout", "dq", "dk", "dv", "ws"):
            setattr(a, n, 4096)
        a.ws_bytes = 1 << 60
        assert L["sar_xattn_fwd_" + sfx](ctypes.byref(a), None) == -1 and L["sar_xattn_bwd_" + sfx](ctypes.byref(a), None) == -1, kw
        assert L["sar_kv8_attend_" + sfx](ctypes.byref(a), 4096, 4096, 4096, 4096, 1 << 20, None) == -1, kw
        assert L["sar_xattn_fwd_workspace_bytes"](ctypes.byref(a)) == 0


def test_a_status_for_bad_arguments_is_a_value_error(monkeypatch):
    from aesrc2020_amd import _lib, attention

    class Device:
        index = 0
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    for status, error in ((-1, ValueError), (-2, RuntimeError)):
        monkeypatch.setitem(_lib.lib().fn, "sar_nothing", lambda *a, s=status: s)
        with pytest.raises(error):
            attention._launch("sar_nothing", Device())
