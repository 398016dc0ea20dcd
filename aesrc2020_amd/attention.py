"""Attention of decoder tokens to the encoder's states (csrc/xattn.hip, csrc/xattn_step.hip): the operators an attention decoder needs beside
the CTC branch (model.py:117-119).  cross_attention / cross_attention_grad are the training pair, cross_attention with one row per utterance
is the single-token form, EncoderCache8 holds an utterance's keys and values in 8 bits and attends to them.

Everything runs on the current HIP stream of the tensors' device, allocates through torch (so calls can be captured into a HIP graph) and
raises ValueError for arguments it does not take.  layers.CrossAttention is the Layer over the same calls."""
import ctypes
import struct

import torch

from . import _lib
from ._call import SFX as _SFX, given as _given, launch as _launch, result as _result, with_workspace as _place

_P, _L, _I = ctypes.c_void_p, ctypes.c_long, ctypes.c_int


class Xattn(ctypes.Structure):
    """include/sarnet.h: sarXattn."""
    _fields_ = [(n, _P) for n in ("q", "k", "v", "dout", "out", "lse", "dq", "dk", "dv", "k_lens", "q_lens", "ws")] + [("ws_bytes", _L)] + \
               [(n, _L) for n in ("q_sb", "q_st", "q_sh", "k_sb", "k_st", "k_sh", "v_sb", "v_st", "v_sh", "o_sb", "o_st", "o_sh", "g_sb", "g_st", "g_sh")] + \
               [(n, _I) for n in ("B", "Tq", "Tk", "Hq", "Hkv", "D")] + [("scale", ctypes.c_float), ("elt_bytes", _I)]


_XATTN = struct.Struct("12Ql15l6ifi")                                  # the same fields: packing bytes costs a fifth of filling the Structure
_WS_AT = Xattn.ws.offset
_NAMES = {n: {d: "sar_%s_%s" % (n, s) for d, s in _SFX.items()} for n in ("xattn_fwd", "xattn_bwd", "kv8_attend")}


def _rows(name, x, like=None):
    """x as the kernels take it: 4-D, last axis contiguous, rows on 16-byte boundaries and at most 16 MB apart -- a view that is not is copied."""
    if x is None:
        raise ValueError("%s is missing" % name)
    if x.dim() != 4:
        raise ValueError("%s has to be (batch, time, heads, dim), got shape %r" % (name, tuple(x.shape)))
    if like is None:
        if x.dtype not in _SFX:
            raise ValueError("%s has to be float32, bfloat16 or float16, got %s" % (name, x.dtype))
        if not x.is_cuda:
            raise ValueError("%s is on %s: the kernels need a HIP device, there is no CPU fallback" % (name, x.device))
    elif x.dtype != like.dtype or x.device != like.device:
        raise ValueError("%s is %s on %s, the queries are %s on %s" % (name, x.dtype, x.device, like.dtype, like.device))
    sb, st, sh, sd = x.stride()
    if sd != 1 and x.shape[3] != 1 or (sb | st | sh) * x.element_size() & 15 or x.data_ptr() & 15 or st > 1 << 22:
        return x.clone(memory_format=torch.contiguous_format)          # (a fresh allocation is aligned; contiguous() may hand x back)
    return x


def _lens(name, lens, B, device):
    if lens is None:
        return 0
    if lens.dtype != torch.int32 or lens.shape != (B,) or lens.device != device or not lens.is_contiguous():
        raise ValueError("%s has to be a contiguous int32 tensor of %d lengths on %s" % (name, B, device))
    return lens.data_ptr()


def _heads(Hq, Hkv, D):
    if Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise ValueError("%d query heads are not a multiple of %d key heads" % (Hq, Hkv))
    if D % 8 or not 8 <= D <= 128:
        raise ValueError("the head width has to be a multiple of 8 from 8 to 128, got %d" % D)


def _with_workspace(query, device, a):
    """sarXattn as bytes -> the same with a workspace where the call needs one, and the workspace to keep until the launch."""
    n = _lib.lib().fn[query](a)
    if not n:
        return a, None
    ws = torch.empty(n, dtype=torch.uint8, device=device)
    return _place(a, _WS_AT, ws), ws


def _result_like(name, t, q):
    """`t`, or a new tensor, of q's shape and type, contiguous (empty_like is the faster call; q's rows are aligned: _rows)."""
    return torch.empty_like(q) if t is None and q.is_contiguous() else _result(name, t, q.shape, q.dtype, q.device)


def _scale(scale, D):
    return D ** -0.5 if scale is None else float(scale)


def _check_kv(q, k, v):
    k, v = _rows("k", k, q), _rows("v", v, q)
    ks, qs = k.shape, q.shape
    if ks != v.shape or ks[0] != qs[0] or ks[3] != qs[3]:
        raise ValueError("q %r, k %r and v %r do not fit" % (tuple(qs), tuple(ks), tuple(v.shape)))
    _heads(qs[2], ks[2], qs[3])
    return k, v


def cross_attention(q, k, v, k_lens=None, q_lens=None, scale=None, return_lse=False, out=None, lse=None):
    """softmax(scale q k^T) v over each utterance's first k_lens frames.

    q (B, Tq, Hq, D), k, v (B, Tk, Hkv, D), Hq a multiple of Hkv (query head h reads key head h // (Hq // Hkv)); fp32, bf16 or fp16; any
    strides whose last is 1.  k_lens, q_lens: int32 (B,) or None.  scale: 1 / sqrt(D) if None.  -> out (B, Tq, Hq, D), and with return_lse the rows'
    log-sum-exp (B, Hq, Tq) fp32 that cross_attention_grad needs.  Rows from q_lens on and rows of an utterance without frames are
    zeros (lse -inf); frames from k_lens on are not looked at.  `out`, `lse`: buffers to write into."""
    q = _rows("q", q)
    k, v = _check_kv(q, k, v)
    B, Tq, Hq, D = q.shape
    Tk, Hkv, device = k.shape[1], k.shape[2], q.device
    out = _result_like("out", out, q)
    if return_lse or lse is not None:
        lse = _result("lse", lse, (B, Hq, Tq), torch.float32, device)
    kl = 0 if k_lens is None else _lens("k_lens", k_lens, B, device)
    ql = 0 if q_lens is None else _lens("q_lens", q_lens, B, device)
    if B and Tq:
        qp, sq, sk, sv = q.data_ptr(), q.stride(), k.stride(), v.stride()
        a = _XATTN.pack(qp, k.data_ptr() if Tk else qp, v.data_ptr() if Tk else qp, 0, out.data_ptr(), 0 if lse is None else lse.data_ptr(), 0, 0, 0, kl, ql, 0, 0,      # (no frames: never read)
                        sq[0], sq[1], sq[2], sk[0], sk[1], sk[2], sv[0], sv[1], sv[2], Tq * Hq * D, Hq * D, D, 0, 0, 0, B, Tq, Tk, Hq, Hkv, D, _scale(scale, D), q.element_size())
        if Tk > 256:                                                   # (sarnet.h: 256 keys never need a workspace)
            a, ws = _with_workspace("sar_xattn_fwd_workspace_bytes", device, a)
        _launch(_NAMES["xattn_fwd"][q.dtype], device, a)
    return (out, lse) if return_lse else out


def cross_attention_grad(dout, q, k, v, out, lse, k_lens=None, q_lens=None, scale=None, dq=None, dk=None, dv=None):
    """Gradients of cross_attention: dout as out, the other arguments as the forward took and gave them -> (dq, dk, dv), contiguous, of the
    inputs' type (each element rounded once from an fp32 sum; the gradient of a key head is the sum over its query heads).  No atomics: the
    same inputs give the same bits.  `dq`, `dk`, `dv`: buffers to write into."""
    q = _rows("q", q)
    k, v = _check_kv(q, k, v)
    dout, out = _rows("dout", dout, q), _rows("out", out, q)
    B, Tq, Hq, D = q.shape
    Tk, Hkv, device = k.shape[1], k.shape[2], q.device
    if dout.shape != q.shape or out.shape != q.shape:
        raise ValueError("dout %r and out %r have to have the shape of q %r" % (tuple(dout.shape), tuple(out.shape), tuple(q.shape)))
    lse = _given("lse", lse, (B, Hq, Tq), torch.float32, device)
    dq = _result_like("dq", dq, q) if B and Tq else _result("dq", dq, q.shape, q.dtype, device)
    dk, dv = _result("dk", dk, k.shape, q.dtype, device), _result("dv", dv, v.shape, q.dtype, device)
    kl = 0 if k_lens is None else _lens("k_lens", k_lens, B, device)
    ql = 0 if q_lens is None else _lens("q_lens", q_lens, B, device)
    if Tq == 0:
        dk.zero_(); dv.zero_()
    elif B:
        qp, sq, sk, sv, so, sg = q.data_ptr(), q.stride(), k.stride(), v.stride(), out.stride(), dout.stride()
        a = _XATTN.pack(qp, k.data_ptr() if Tk else qp, v.data_ptr() if Tk else qp, dout.data_ptr(), out.data_ptr(), lse.data_ptr(), dq.data_ptr(),
                        dk.data_ptr() if Tk else qp, dv.data_ptr() if Tk else qp, kl, ql, 0, 0,  # (no frames: never read or written)
                        sq[0], sq[1], sq[2], sk[0], sk[1], sk[2], sv[0], sv[1], sv[2], so[0], so[1], so[2], sg[0], sg[1], sg[2], B, Tq, Tk, Hq, Hkv, D, _scale(scale, D), q.element_size())
        a, ws = _with_workspace("sar_xattn_bwd_workspace_bytes", device, a)
        _launch(_NAMES["xattn_bwd"][q.dtype], device, a)
    return dq, dk, dv


class EncoderCache8:
    """An utterance batch's keys and values in 8 bits for decoding token by token: half (a quarter) of the bytes of 16-bit (fp32) ones, and every
    token reads all of them.

    k8, v8 (batch, heads, frames rounded up to 64, dim) float8_e4m3fn; k_scale, v_scale (batch, heads, blocks of 64 frames) fp32 powers of two,
    value = e4m3 * scale; lens (batch,) int32.  The buffers keep their addresses for the cache's life, so a captured step stays valid over store().
    stored: frames that store() has written, in whole blocks, which the next chunk may start at (to be set where the buffers are filled otherwise)."""

    BLOCK = 64

    def __init__(self, batch, frames, heads, dim, device="cuda"):
        batch, frames, heads, dim = int(batch), int(frames), int(heads), int(dim)
        _heads(heads, heads, dim)
        if batch < 1 or frames < 1:
            raise ValueError("a cache needs at least one utterance and one frame, got %d and %d" % (batch, frames))
        self.batch, self.frames, self.heads, self.dim = batch, frames, heads, dim
        n = -(-frames // self.BLOCK)
        self.k8, self.v8 = (torch.empty(batch, heads, n * self.BLOCK, dim, dtype=torch.float8_e4m3fn, device=device) for _ in range(2))
        self.k_scale, self.v_scale = (torch.empty(batch, heads, n, dtype=torch.float32, device=device) for _ in range(2))
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)                         # (nothing behind a length is ever read)
        self.device = self.k8.device
        self.stored = 0

    def store(self, k, v, k_lens=None, first=0):
        """Write frames [first, first + T) of every utterance from k, v (batch, T, heads, dim) (fp32, bf16 or fp16); `first` is a multiple of 64:
        a streaming encoder appends chunks, all but an utterance's last of whole blocks.  k_lens: how many of these T frames each utterance has (int32 (batch,); None: all) -- the
        rest is stored as zeros.  The cache's lens become first + k_lens; with first > 0 an utterance without new frames keeps its length."""
        k, v = _rows("k", k), _rows("v", v, k)
        B, T, H, D = k.shape
        if k.shape != v.shape or B != self.batch or H != self.heads or D != self.dim or k.device != self.device:
            raise ValueError("k %r and v %r on %s do not fit a cache of %d utterances, %d heads of %d on %s" %
                             (tuple(k.shape), tuple(v.shape), k.device, self.batch, self.heads, self.dim, self.device))
        first = int(first)
        if first < 0 or first % self.BLOCK or T < 1 or first + T > self.frames:
            raise ValueError("frames [%d, %d) do not fit: first has to be a multiple of %d, the cache has %d frames" % (first, first + T, self.BLOCK, self.frames))
        if first > self.stored:
            raise ValueError("frames [%d, %d) were never stored: a chunk starts where the ones before it end" % (self.stored, first))
        kl = _lens("k_lens", k_lens, B, k.device)
        _launch("sar_kv8_store_" + _SFX[k.dtype], k.device, k.data_ptr(), *k.stride()[:3], v.data_ptr(), *v.stride()[:3], kl, self.k8.data_ptr(), self.k_scale.data_ptr(),
                self.v8.data_ptr(), self.v_scale.data_ptr(), self.lens.data_ptr(), B, T, H, D, self.k8.shape[2], first)
        self.stored = -(-(first + T) // self.BLOCK) * self.BLOCK

    def attend(self, q, q_lens=None, scale=None, out=None):
        """cross_attention(q, held k, held v, k_lens=lens): q (batch, Tq, Hq, dim) of any of the three types, Hq a multiple of the cache's heads
        -> out of q's type.  Made for a few rows (Tq Hq / heads); each 32 of them read the cache once."""
        q = _rows("q", q)
        B, Tq, Hq, D = q.shape
        device = q.device
        if B != self.batch or D != self.dim or device != self.device:
            raise ValueError("q %r on %s does not fit a cache of %d utterances, %d heads of %d on %s" % (tuple(q.shape), device, self.batch, self.heads, self.dim, self.device))
        if Hq < 1 or Hq % self.heads:
            _heads(Hq, self.heads, D)
        out = _result_like("out", out, q)
        ql = 0 if q_lens is None else _lens("q_lens", q_lens, B, device)
        if Tq:
            s = q.stride()
            a = _XATTN.pack(q.data_ptr(), 0, 0, 0, out.data_ptr(), 0, 0, 0, 0, self.lens.data_ptr(), ql, 0, 0, s[0], s[1], s[2], 0, 0, 0, 0, 0, 0, Tq * Hq * D, Hq * D, D, 0, 0, 0,
                            B, Tq, self.frames, Hq, self.heads, D, _scale(scale, D), q.element_size())
            if self.frames > 256:
                a, ws = _with_workspace("sar_kv8_attend_workspace_bytes", device, a)
            _launch(_NAMES["kv8_attend"][q.dtype], device, a, self.k8.data_ptr(), self.k_scale.data_ptr(), self.v8.data_ptr(), self.v_scale.data_ptr(), self.k8.shape[2])
        return out
