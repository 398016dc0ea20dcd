"""What the calls of the decoder operators (attention.py, losses.py) share: element types, checks of buffers, the launch."""
import struct

import torch

from . import _lib

SFX = {torch.float32: "f32", torch.bfloat16: "bf16", torch.float16: "f16"}        # the entry points' suffixes
_WS = struct.Struct("Ql")                                              # {ws, ws_bytes} of an argument struct


def launch(name, device, *args):
    """Call an entry point on the current stream of the tensors' device."""
    fn = _lib.lib().fn[name]
    index = device.index
    if torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            rc = fn(*args, torch.cuda.current_stream().cuda_stream)
    else:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))      # (torch.cuda.current_stream().cuda_stream without the Stream object: 2 us less)
    if rc == -1:
        raise ValueError("%s does not take these arguments: include/sarnet.h states its limits" % name)
    if rc != 0:
        raise RuntimeError("%s failed with status %d" % (name, rc))


def result(name, t, shape, dtype, device):
    if t is None:
        return torch.empty(shape, dtype=dtype, device=device)
    if tuple(t.shape) != tuple(shape) or t.dtype != dtype or t.device != device or not t.is_contiguous() or t.data_ptr() % 16:
        raise ValueError("%s has to be a contiguous, 16-byte aligned %s tensor of shape %r on %s" % (name, dtype, tuple(shape), device))
    return t


def given(name, t, shape, dtype, device):
    """An fp32 vector that a gradient reads as it is: lse, dloss."""
    if t is None or tuple(t.shape) != tuple(shape) or t.dtype != dtype or t.device != device or not t.is_contiguous():
        raise ValueError("%s has to be a contiguous %s tensor of shape %r on %s, got %s" %
                         (name, dtype, tuple(shape), device, "None" if t is None else "%s %r on %s" % (t.dtype, tuple(t.shape), t.device)))
    return t


def with_workspace(a, at, ws):
    """The bytes of an argument struct with the workspace `ws` at offset `at`."""
    return a[:at] + _WS.pack(ws.data_ptr(), ws.numel()) + a[at + _WS.size:]
