"""Margin-softmax heads and circle loss, MI355X-native (mirrors /root/reference/losses.py).

SphereFace / CosFace / ArcFace keep the reference constructor (n_classes, s, m, regularizer) and call convention
`layer([x, y_onehot]) -> softmax probabilities` (losses.py:28-47, 74-91, 121-144); weight `W (D, n_classes)`,
glorot_uniform (losses.py:22-26).  circle_loss(y_true, y_pred, gamma, margin) -> per-sample loss (losses.py:157-172).
"""
import ctypes
import struct

import torch

from . import _lib
from ._call import SFX as _SFX, given as _given, launch as _launch, result as _result, with_workspace
from .engine import glorot_uniform
from .layers import Layer

_call = _lib.call


class _MarginHead(Layer):
    MODE = None

    def __init__(self, n_classes=10, s=30.0, m=None, regularizer=None, name=None, in_dim=None, **kwargs):
        super().__init__(name or self.__class__.__name__.lower())
        self.n_classes, self.s, self.m = int(n_classes), float(s), float(self.DEFAULT_M if m is None else m)
        self.l2 = float(regularizer) if regularizer else 0.0      # reference passes regularizer=None
        self.W = None
        if in_dim is not None:
            self.build(in_dim)

    def build(self, in_dim):
        A = self.n_classes
        self.W = self.store.add(self.name + "/W", (in_dim, A), glorot_uniform(self.store.rng, (in_dim, A), in_dim, A), self.l2)
        self.D = in_dim
        self.output_shape = (None, A)

    def compute_output_shape(self, input_shape):
        return (None, self.n_classes)

    def __call__(self, inputs):
        return self.forward(*inputs)

    def forward(self, x, y):
        B, D, A = x.shape[0], self.D, self.n_classes
        self.x, self.y, self.B = x, y, B
        self.probs = self.buf("probs", (B, A)); self.cosv = self.buf("cos", (B, A))
        self.inv_x = self.buf("inv_x", (B,)); self.inv_w = self.buf("inv_w", (A,))
        _call("sar_margin_head_fwd_f32", x, y, self.W.w, self.probs, self.cosv, self.inv_x, self.inv_w, B, D, A, self.MODE, self.s, self.m)
        return self.probs

    def train(self, x, y, y_true, dloss, dx_out, accumulate_dx=False):
        """forward + categorical_crossentropy(y_true, probs) + backward of both in two launches (csrc/heads.hip: margin_train_kernel):
        -> (probs, per-sample loss); dx_out written / accumulated, W.g accumulated."""
        B, D, A = x.shape[0], self.D, self.n_classes
        self.x, self.y, self.B = x, y, B
        self.probs = self.buf("probs", (B, A)); self.inv_w = self.buf("inv_w", (A,)); loss = self.buf("loss", (B,))
        key = self.name + "/dwn_ws"
        fresh = key not in self.store.bufs.d
        ws = self.buf("dwn_ws", (D, A))
        if fresh:
            ws.zero_()                                             # the kernels keep it zero from here on (first step is eager)
        _call("sar_margin_head_train_f32", x, y, y_true, dloss, self.W.w, self.probs, loss, self.inv_w, dx_out, self.W.g, ws, B, D, A,
              self.MODE, self.s, self.m, 1 if accumulate_dx else 0)
        return self.probs, loss

    def train_buffers(self, x, y, B):
        """Buffers of the training step when another launch runs it (model.py: sar_accent_margin_train_f32): -> (workspace of D*A + 1
        words the kernel keeps zero, probs, per-sample loss, inv_w)."""
        D, A = self.D, self.n_classes
        self.x, self.y, self.B = x, y, B
        self.probs = self.buf("probs", (B, A)); self.inv_w = self.buf("inv_w", (A,))
        key = self.name + "/dwn_ws1"
        fresh = key not in self.store.bufs.d
        ws = self.buf("dwn_ws1", (D * A + 1,))
        if fresh:
            ws.zero_()
        return ws, self.probs, self.buf("loss", (B,)), self.inv_w

    def backward(self, dprobs, dx_out=None, accumulate_dx=False):
        B, D, A = self.B, self.D, self.n_classes
        dx = dx_out if dx_out is not None else self.buf("dx", (B, D))
        ws = self.buf("dwn_ws_bwd", (D, A))
        _call("sar_margin_head_bwd_f32", dprobs, self.probs, self.cosv, self.x, self.y, self.W.w, self.inv_x, self.inv_w, dx,
              self.W.g, ws, B, D, A, self.MODE, self.s, self.m, 1 if accumulate_dx else 0)
        return dx


class SphereFace(_MarginHead):
    MODE, DEFAULT_M = 0, 1.35


class CosFace(_MarginHead):
    MODE, DEFAULT_M = 1, 0.35


class ArcFace(_MarginHead):
    MODE, DEFAULT_M = 2, 0.50


class CircleLoss:
    """Callable with the reference's signature plus an explicit backward (the reference relies on TF autodiff)."""

    def __init__(self, bufs, key="circle"):
        self.bufs, self.key = bufs, key

    def forward(self, y_true, y_pred, gamma=256, margin=0.25):
        B, A = y_pred.shape
        self.y, self.s, self.gamma, self.margin = y_true, y_pred, float(gamma), float(margin)
        self.loss = self.bufs.get(self.key + "/loss", (B,))
        _call("sar_circle_loss_fwd_f32", y_true, y_pred, self.loss, B, A, self.gamma, self.margin)
        return self.loss

    def backward(self, dloss):
        B, A = self.s.shape
        ds = self.bufs.get(self.key + "/ds", (B, A))
        _call("sar_circle_loss_bwd_f32", self.y, self.s, dloss, ds, B, A, self.gamma, self.margin)
        return ds


def circle_loss(y_true, y_pred, gamma=256, margin=0.25):
    """losses.py:157-172 (forward only; SAR_Net uses CircleLoss for the train step)."""
    import torch
    B, A = y_pred.shape
    loss = torch.empty(B, dtype=torch.float32, device=y_pred.device)
    _call("sar_circle_loss_fwd_f32", y_true, y_pred, loss, B, A, float(gamma), float(margin))
    return loss


class CategoricalCrossentropy:
    """Keras categorical_crossentropy on probabilities (model.py:350,354) with explicit backward."""

    def __init__(self, bufs, key):
        self.bufs, self.key = bufs, key

    def forward(self, y_true, p):
        B, A = p.shape
        self.y, self.p = y_true, p
        self.loss = self.bufs.get(self.key + "/loss", (B,))
        _call("sar_cce_fwd_f32", y_true, p, self.loss, B, A)
        return self.loss

    def backward(self, dloss):
        B, A = self.p.shape
        dp = self.bufs.get(self.key + "/dp", (B, A))
        _call("sar_cce_bwd_f32", self.y, self.p, dloss, dp, B, A)
        return dp


# ---- softmax cross entropy over a vocabulary, from the hidden rows and the output layer's kernel (csrc/vocab_ce.hip)
class _VocabCe(ctypes.Structure):
    """include/sarnet.h: sarVocabCe."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("x", "kernel", "bias", "labels", "dloss", "loss", "lse", "dx", "dkernel", "dbias", "ws")] + \
               [(n, ctypes.c_long) for n in ("ws_bytes", "ldx", "ldk")] + [(n, ctypes.c_int) for n in ("R", "D", "V", "label_bytes", "accumulate", "pad_")]


_VOCAB_CE = struct.Struct("11Q3l6i")                                        # the same fields as bytes
_WS_AT = _VocabCe.ws.offset
_LABELS = {torch.int32: 4, torch.int64: 8}


def _vocab_args(x, kernel, labels, bias):
    """-> x, kernel (rows contiguous), R, D, V: as the kernels take them."""
    if x is None or kernel is None or labels is None:
        raise ValueError("x, kernel and labels have to be given")
    xs, ks = x.shape, kernel.shape
    if len(xs) != 2 or len(ks) != 2 or xs[1] != ks[0] or ks[0] < 1 or ks[1] < 1:
        raise ValueError("x %r and kernel %r have to be (rows, D) and (D, vocabulary)" % (tuple(xs), tuple(ks)))
    R, D, V = xs[0], ks[0], ks[1]
    dtype, device = x.dtype, x.device
    if dtype not in _SFX or not x.is_cuda:
        raise ValueError("x has to be a float32, bfloat16 or float16 tensor on a HIP device, got %s on %s" % (dtype, device))
    if kernel.dtype != dtype or kernel.device != device:
        raise ValueError("kernel is %s on %s, x is %s on %s" % (kernel.dtype, kernel.device, dtype, device))
    if bias is not None and (bias.shape != (V,) or bias.dtype != dtype or bias.device != device or not bias.is_contiguous()):
        raise ValueError("bias has to be a contiguous %s tensor of %d values on %s" % (dtype, V, device))
    if labels.shape != (R,) or labels.dtype not in _LABELS or labels.device != device or not labels.is_contiguous():
        raise ValueError("labels have to be a contiguous int32 or int64 tensor of %d values on %s" % (R, device))
    if R > 1 << 22 or V > 1 << 22 or D > 1 << 16 or (R // 64 + 1) * (V // 64 + 1) > 1 << 28:
        raise ValueError("%d rows, %d wide, over %d classes: at most 2^22, 2^16 and 2^22 are taken, and 2^40 logits" % (R, D, V))
    step, one = x.stride()
    if R and (one != 1 or not D <= step <= 1 << 22):
        x = x.clone(memory_format=torch.contiguous_format)
    step, one = kernel.stride()
    if one != 1 or not V <= step <= 1 << 22:
        kernel = kernel.clone(memory_format=torch.contiguous_format)
    return x, kernel, R, D, V


def _vocab_launch(direction, x, kernel, labels, bias, dloss, loss, lse, dx, dkernel, dbias, R, D, V, accumulate=0):
    dtype, device = x.dtype, x.device
    name = "sar_vocab_ce_%s_%s" % (direction, _SFX[dtype])
    args = (x.data_ptr(), kernel.data_ptr(), _ptr(bias), labels.data_ptr(), _ptr(dloss), _ptr(loss), _ptr(lse), _ptr(dx), _ptr(dkernel), _ptr(dbias), 0, 0,
            x.stride(0) if R > 1 else D, kernel.stride(0) if D > 1 else V, R, D, V, _LABELS[labels.dtype], accumulate, 0)
    a = _VOCAB_CE.pack(*args)
    n = _lib.lib().fn[name + "_workspace_bytes"](a)
    ws = torch.empty(n, dtype=torch.uint8, device=device)                    # (torch's blocks are 512-byte aligned)
    _launch(name, device, with_workspace(a, _WS_AT, ws))


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def vocab_crossentropy(x, kernel, labels, bias=None, return_lse=False, loss=None, lse=None):
    """-log softmax(x @ kernel + bias)[label] of every row, without keeping the logits.

    x (R, D) hidden rows, kernel (D, V) in the Dense layout, bias (V) or None: all fp32, bf16 or fp16; labels (R) int32 or int64, a label outside
    [0, V) leaves its row out (loss 0).  -> loss (R) fp32, and with return_lse the rows' log-sum-exp (R) fp32 that vocab_crossentropy_grad needs."""
    x, kernel, R, D, V = _vocab_args(x, kernel, labels, bias)
    loss = _result("loss", loss, (R,), torch.float32, x.device)
    if return_lse or lse is not None:
        lse = _result("lse", lse, (R,), torch.float32, x.device)
    if R:
        _vocab_launch("fwd", x, kernel, labels, bias, None, loss, lse, None, None, None, R, D, V)
    return (loss, lse) if return_lse else loss


def vocab_crossentropy_grad(dloss, x, kernel, labels, lse, bias=None, dx=None, dkernel=None, dbias=None, accumulate=False, need_dx=True):
    """Gradients of vocab_crossentropy: dloss (R) fp32 -> (dx, dkernel, dbias | None) of the inputs' type, each element rounded once from an fp32
    sum.  accumulate (fp32 only): add to the `dkernel`, `dbias` given, as parameter gradients of this package are.  need_dx=False: dx is None.
    softmax - onehot is held in 16 bits (fp32: about twice that).  A row's dx does not depend on other rows, but for fp16, where those bits are relative
    to the largest |dloss| of a row with a label: such rows of very different dloss (2^20 and more) belong in different calls.  dkernel, the rows' sum, is
    good to 2^-38 of the largest |x dloss| (fp32 and bf16, larger calls).  x has to be finite in rows that are left out too.
    No atomics: the same inputs give the same bits."""
    x, kernel, R, D, V = _vocab_args(x, kernel, labels, bias)
    if accumulate and (x.dtype != torch.float32 or dkernel is None or (bias is not None and dbias is None)):
        raise ValueError("accumulate needs fp32 and the buffers to add to")
    dloss, lse = _given("dloss", dloss, (R,), torch.float32, x.device), _given("lse", lse, (R,), torch.float32, x.device)
    dx = _result("dx", dx, (R, D), x.dtype, x.device) if need_dx else None
    dkernel = _result("dkernel", dkernel, (D, V), x.dtype, x.device)
    dbias = None if bias is None else _result("dbias", dbias, (V,), x.dtype, x.device)
    if R:
        _vocab_launch("bwd", x, kernel, labels, bias, dloss, None, lse, dx, dkernel, dbias, R, D, V, 1 if accumulate else 0)
    elif not accumulate:
        dkernel.zero_()
        if dbias is not None:
            dbias.zero_()
    return dx, dkernel, dbias


class VocabCrossentropy:
    """Softmax layer + cross entropy of a label-synchronous branch as one object with explicit backward: what Dense(..., "softmax") followed by
    CategoricalCrossentropy computes, for the weights of a Dense layer (bias or none) and integer labels."""

    def __init__(self, bufs, key, dense):
        self.bufs, self.key, self.dense = bufs, key, dense

    def forward(self, x, labels):
        R = x.numel() // self.dense.in_dim
        self.x, self.labels = x.view(R, self.dense.in_dim), labels
        self.bias = None if self.dense.bias is None else self.dense.bias.w
        self.loss, self.lse = self.bufs.get(self.key + "/loss", (R,)), self.bufs.get(self.key + "/lse", (R,))
        vocab_crossentropy(self.x, self.dense.kernel.w, labels, self.bias, True, self.loss, self.lse)
        return self.loss

    def backward(self, dloss, need_dx=True):
        """-> dx; the layer's kernel and bias gradients are accumulated."""
        dx = self.bufs.get(self.key + "/dx", tuple(self.x.shape)) if need_dx else None
        vocab_crossentropy_grad(dloss, self.x, self.dense.kernel.w, self.labels, self.lse, self.bias, dx, self.dense.kernel.g,
                                None if self.bias is None else self.dense.bias.g, accumulate=True, need_dx=need_dx)
        return dx
