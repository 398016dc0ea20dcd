"""Attention and the 8-bit cache in float64 for the tests: the definitions, row by row."""
import math

import torch


def attend(q, k, v, k_lens=None, q_lens=None, scale=None, dout=None):
    """q (B, Tq, Hq, D), k, v (B, Tk, Hkv, D) -> (out, lse) or (out, lse, dq, dk, dv), float64.  Frames behind a length are never touched, rows behind a
    length and rows without frames give zeros (lse -inf)."""
    B, Tq, Hq, D = q.shape
    Tk, Hkv = k.shape[1], k.shape[2]
    G = Hq // Hkv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    q, k, v = q.double(), k.double(), v.double()
    out = torch.zeros_like(q)
    lse = torch.full((B, Hq, Tq), -math.inf, dtype=torch.float64, device=q.device)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b in range(B):
        n = Tk if k_lens is None else max(0, min(Tk, int(k_lens[b])))
        m = Tq if q_lens is None else max(0, min(Tq, int(q_lens[b])))
        if n == 0 or m == 0:
            continue
        for h in range(Hq):
            qq, kk, vv = q[b, :m, h], k[b, :n, h // G], v[b, :n, h // G]
            s = scale * (qq @ kk.T)
            top = s.max(1, keepdim=True).values
            e = torch.exp(s - top)
            tot = e.sum(1, keepdim=True)
            p = e / tot
            out[b, :m, h] = p @ vv
            lse[b, h, :m] = (top + torch.log(tot))[:, 0]
            if dout is not None:
                g = dout[b, :m, h].double()
                dp = g @ vv.T
                ds = p * (dp - (p * dp).sum(1, keepdim=True))
                dq[b, :m, h] = scale * (ds @ kk)
                dk[b, :n, h // G] += scale * (ds.T @ qq)
                dv[b, :n, h // G] += p.T @ g
    return (out, lse) if dout is None else (out, lse, dq, dk, dv)


def quantise(x, lens=None, block=64):
    """x (B, T, H, D) -> (e4m3 values as float64 (B, H, N * 64, D), scales (B, H, N) float64).  Computed on the CPU: a GPU's float64 power of two is
    not always the power of two."""
    dev, x = x.device, x.cpu()
    B, T, H, D = x.shape
    N = -(-T // block)
    y = torch.zeros(B, H, N * block, D, dtype=torch.float64, device=x.device)
    y[:, :, :T] = x.double().transpose(1, 2)
    if lens is not None:
        for b in range(B):
            y[b, :, max(0, min(T, int(lens[b]))):] = 0
    y = y.view(B, H, N, block, D)
    fin = torch.where(torch.isfinite(y), y.abs(), torch.zeros_like(y)).amax((3, 4))
    s = torch.ones_like(fin)
    for i in (fin > 0).nonzero().tolist():
        top = float(fin[tuple(i)])
        m, e = math.frexp(top)
        s[tuple(i)] = 2.0 ** max(e - 9 if m <= 0.875 else e - 8, -118)
    z = y / s[..., None, None]
    step = 2.0 ** (torch.floor(torch.log2(z.abs().clamp_min(2.0 ** -6))) - 3)
    z = torch.where(torch.isfinite(z), torch.round(z / step) * step, torch.full_like(z, math.nan))
    return z.reshape(B, H, N * block, D).to(dev), s.to(dev)
