"""Cross attention and the 8-bit key / value cache on the GPU against the float64 definitions (tests/_attn_ref.py).

Tolerances.  u = half a step of the type (finfo.eps / 2: bf16 2^-8, fp16 2^-11, fp32 2^-24).
  out: the kernel rounds the probabilities to the type (relative u each) and the result once (u of the value): |err| <= u (sum_j p_j |v_j| + |out|) plus fp32
  sums and the exponential: the score's fp32 error (about D products summed, 2^-24 (8 + |s| + sum |q k| / 8) in absolute terms) is a relative error
  of p.  sum_j p_j |v_j| <= max |v|.  For fp32 only the second part is there.
  dq, dk, dv: the same argument per product: probabilities and ds are rounded to the type before they meet k, q, do; delta is a sum over the ROUNDED out.
  Each bound below is that arithmetic with the sums of magnitudes evaluated in float64 next to the oracle (attend_abs)."""
import math

import pytest
import torch

from aesrc2020_amd import _lib
from tests import _attn_ref as R

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _att():
    from aesrc2020_amd import attention
    return attention


def u(dt):
    return torch.finfo(dt).eps / 2


def bounds(q, k, v, k_lens, q_lens, scale, dout=None):
    """Elementwise bounds of |kernel - float64| from the module's derivation."""
    dt = q.dtype
    B, Tq, Hq, D = q.shape
    Tk, Hkv = k.shape[1], k.shape[2]
    G = Hq // Hkv
    uu = u(dt) if dt != torch.float32 else 0.0
    f = 2.0 ** -24
    q, k, v = q.double(), k.double(), v.double()
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    ro = u(dt)                                                     # the result's own rounding
    eo = torch.zeros_like(q); eq = torch.zeros_like(q); ek = torch.zeros_like(k); ev = torch.zeros_like(v)
    for b in range(B):
        n = Tk if k_lens is None else max(0, min(Tk, int(k_lens[b])))
        m = Tq if q_lens is None else max(0, min(Tq, int(q_lens[b])))
        if n == 0 or m == 0:
            continue
        for h in range(Hq):
            qq, kk, vv = q[b, :m, h], k[b, :n, h // G], v[b, :n, h // G]
            s = scale * (qq @ kk.T)
            p = torch.softmax(s, 1)
            # fp32 error of a score: D products accumulated in fp32, the multiplication by scale log2 e, the subtraction of the maximum, exp2; twice
            # for the normaliser (lse has the same error)
            se = f * (D * abs(scale) * (qq.abs() @ kk.abs().T) + 4 * s.abs() + 4 * s.abs().amax(1, keepdim=True) + 16)
            rp = uu + 2 * se + f * (n + 16)                        # relative error of a probability as an operand, and of a sum over n of them
            out = p @ vv
            eo[b, :m, h] = (rp * p) @ vv.abs() + f * n * (p @ vv.abs()) + ro * out.abs()
            if dout is not None:
                g = dout[b, :m, h].double()
                dp = g @ vv.T
                dl = (p * dp).sum(1, keepdim=True)
                ed = (g.abs() * eo[b, :m, h]).sum(1, keepdim=True) + f * D * (g.abs() * out.abs()).sum(1, keepdim=True)      # delta, from the rounded out
                ep = f * D * (g.abs() @ vv.abs().T)
                ds = p * (dp - dl)
                es = (rp + f * 4) * ds.abs() + p * (ep + ed) * (1 + rp)
                eq[b, :m, h] += abs(scale) * (es @ kk.abs() + f * n * (ds.abs() @ kk.abs()))
                ek[b, :n, h // G] += abs(scale) * (es.T @ qq.abs() + f * m * G * (ds.abs().T @ qq.abs()))
                ev[b, :n, h // G] += (rp * p).T @ g.abs() + f * m * G * (p.T @ g.abs())
    if dout is None:
        return eo
    return eo, eq, ek, ev


def check(got, want, bound, what, dt):
    tiny = {torch.float32: 1e-30, torch.bfloat16: 1e-30, torch.float16: 2.0 ** -25}[dt]      # (fp16: half a step of its smallest numbers)
    err = (got.double() - want).abs()
    lim = 1.05 * bound + u(dt) * want.abs() + tiny                 # (1.05: second-order terms)
    assert not torch.isnan(got).any(), what
    worst = (err / lim).max().item() if err.numel() else 0.0
    assert worst <= 1.0, (what, worst, err.max().item())


def make(B, Tq, Tk, Hq, Hkv, D, dt, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dt)  # noqa: E731
    return t(B, Tq, Hq, D), t(B, Tk, Hkv, D), t(B, Tk, Hkv, D), t(B, Tq, Hq, D)


def lens(*a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


#        B, Tq,  Tk, Hq, Hkv, D, k_lens, q_lens
SHAPES = [(1, 1, 1, 1, 1, 8, None, None),
          (1, 1, 39, 4, 4, 64, None, None),
          (2, 1, 300, 6, 2, 72, (300, 33), None),
          (3, 5, 64, 4, 1, 128, (64, 0, 1), (5, 5, 2)),
          (2, 33, 65, 2, 2, 32, (65, 31), (33, 0)),
          (1, 72, 39, 8, 8, 64, None, None),
          (2, 129, 257, 3, 1, 40, (257, 256), (129, 128)),
          (2, 50, 1030, 4, 2, 96, (1030, 700), None),
          (1, 16, 2100, 2, 1, 104, None, None),
          (3, 200, 7, 2, 2, 16, (7, 6, 0), None),
          (1, 9, 1500, 2, 1, 64, None, None),                      # few rows, many keys: dQ in key slices
          (2, 600, 5, 8, 1, 48, (5, 1), (600, 577)),               # few keys, many rows of shared heads: dK, dV in row slices
          (1, 300, 1300, 6, 3, 128, None, None),
          (2, 130, 64, 4, 2, 128, (33, 32), (130, 64)), (3, 65, 33, 2, 2, 96, (33, 0, 2), (0, 65, 64)), (1, 300, 64, 3, 1, 24, None, None),
          (1, 700, 64, 2, 1, 64, None, None)]


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s[:6])))
def test_forward_and_gradients(shape, dt):
    A = _att()
    B, Tq, Tk, Hq, Hkv, D, kl, ql = shape
    q, k, v, g = make(B, Tq, Tk, Hq, Hkv, D, DT[dt], seed=Tk)
    kl, ql = (None if x is None else lens(*x) for x in (kl, ql))
    for i in range(B):                                             # what lies behind a length must not matter
        if kl is not None:
            k[i, int(kl[i]):] = math.nan; v[i, int(kl[i]):] = math.inf
    out, lse = A.cross_attention(q, k, v, k_lens=kl, q_lens=ql, return_lse=True)
    dq, dk, dv = A.cross_attention_grad(g, q, k, v, out, lse, k_lens=kl, q_lens=ql)
    for i in range(B):
        if kl is not None:
            k[i, int(kl[i]):] = 0; v[i, int(kl[i]):] = 0
    want = R.attend(q, k, v, kl, ql, dout=g)
    bd = bounds(q, k, v, kl, ql, None, g)
    check(out, want[0], bd[0], "out", DT[dt])
    fin = torch.isfinite(want[1])
    assert torch.equal(torch.isneginf(lse), ~fin)
    s = want[1][fin].abs().max().item() if fin.any() else 0.0
    assert (lse.double() - want[1])[fin].abs().max().item() <= 2.0 ** -24 * (D * D ** 0.5 * 16 + 8 * s + Tk + 32) if fin.any() else True
    for got, w, e, name in zip((dq, dk, dv), want[2:], bd[1:], ("dq", "dk", "dv")):
        check(got, w, e, name, DT[dt])
    again = A.cross_attention_grad(g, q, k, v, out, lse, k_lens=kl, q_lens=ql)
    assert all(torch.equal(x, y) for x, y in zip((dq, dk, dv), again))


@pytest.mark.parametrize("dt", DT)
def test_one_key_gives_exact_results(dt):
    """One frame (of one, or of many with a length of 1): its probability is 1, the output is v, nothing flows to q and k, dv sums dout.
    The forward takes p = exp2(fma(s, f, -m)) and divides by the sum: with one key p = l = 1 + d, d a few 2^-24, and out = fl(fl(p v) fl(1 / l)): three
    roundings of 2^-24 whatever d is -- fp32 is that near v, and a 16-bit result, whose half step is far wider, is v itself."""
    A = _att()
    q, k, v, g = make(2, 70, 40, 4, 2, 48, DT[dt], seed=12)
    for kk, vv, kl in ((k[:, :1], v[:, :1], None), (k, v, lens(1, 1))):
        out, lse = A.cross_attention(q, kk, vv, k_lens=kl, return_lse=True)
        dq, dk, dv = A.cross_attention_grad(g, q, kk, vv, out, lse, k_lens=kl)
        vv = v[:, :1].repeat_interleave(2, 2).expand(2, 70, 4, 48)
        assert ((out.double() - vv.double()).abs() <= 3.01 * 2.0 ** -24 * vv.double().abs()).all() if dt == "f32" else torch.equal(out, vv)
        assert (dq == 0).all() and (dk == 0).all() and (dv[:, 1:] == 0).all()
        want = g.double().view(2, 70, 2, 2, 48).sum((1, 3))
        assert ((dv[:, 0].double() - want).abs() <= u(DT[dt]) * want.abs() * 1.01 + 2.0 ** -24 * 140 * g.double().abs().view(2, 70, 2, 2, 48).sum((1, 3))).all()


@pytest.mark.parametrize("dt", DT)
def test_gradients_against_differences(dt):
    """d/dt of sum(out * g) along a direction, by central differences of the float64 forward, against the kernels' gradients."""
    A = _att()
    q, k, v, g = make(2, 9, 70, 4, 2, 24, DT[dt], seed=4)
    kl = lens(70, 41)
    out, lse = A.cross_attention(q, k, v, k_lens=kl, return_lse=True)
    grads = A.cross_attention_grad(g, q, k, v, out, lse, k_lens=kl)
    bd = bounds(q, k, v, kl, None, None, g)
    gen = torch.Generator(device="cuda").manual_seed(9)
    for i, (x, dx) in enumerate(zip((q, k, v), grads)):
        w = torch.randn(x.shape, generator=gen, device="cuda", dtype=torch.float64)
        h = 1e-5
        f = [(R.attend(*[(y.double() + (s * h * w if j == i else 0)) for j, y in enumerate((q, k, v))], k_lens=kl)[0] * g.double()).sum() for s in (1, -1)]
        num = ((f[0] - f[1]) / (2 * h)).item()
        ana = (dx.double() * w).sum().item()
        lim = (w.abs() * (1.05 * bd[1 + i] + u(DT[dt]) * dx.double().abs())).sum().item() + 1e-7
        assert abs(num - ana) <= lim, (i, num, ana, lim)


@pytest.mark.parametrize("dt", DT)
def test_strides_orders_and_unaligned_views(dt):
    A = _att()
    t = DT[dt]
    B, Tq, Tk, H, D = 2, 40, 90, 3, 32
    gen = torch.Generator(device="cuda").manual_seed(1)
    kv = torch.randn(B, Tk, 2, H, D, generator=gen, device="cuda").to(t)            # a fused projection's halves
    qh = torch.randn(B, H, Tq, D, generator=gen, device="cuda").to(t)               # head-major
    g = torch.randn(B, Tq, H, D, generator=gen, device="cuda").to(t)
    q, k, v = qh.transpose(1, 2), kv[:, :, 0], kv[:, :, 1]
    raw = torch.randn(B * Tk * H * D + 1, generator=gen, device="cuda").to(t)
    odd = raw[1:].view(B, Tk, H, D)                                # 2 or 4 bytes off a 16-byte boundary
    wide = torch.randn(B, Tk, H, D + 1, generator=gen, device="cuda").to(t)[..., :D]  # rows off it
    for kk, vv in ((k, v), (odd, v), (k, wide), (k[:, :, :1].expand(B, Tk, H, D), v)):
        o1, l1 = A.cross_attention(q, kk, vv, return_lse=True)
        o2, l2 = A.cross_attention(q.contiguous(), kk.contiguous(), vv.contiguous(), return_lse=True)
        assert torch.equal(o1, o2) and torch.equal(l1, l2)
        for x, y in zip(A.cross_attention_grad(g.transpose(1, 2).contiguous().transpose(1, 2), q, kk, vv, o1, l1),
                        A.cross_attention_grad(g, q.contiguous(), kk.contiguous(), vv.contiguous(), o2, l2)):
            assert torch.equal(x, y) and x.is_contiguous()


@pytest.mark.parametrize("dt", DT)
def test_large_scores_given_scale_and_out_buffers(dt):
    """Scores up to about +-600 (a softmax that is one-hot), a negative scale, and results written into given buffers."""
    A = _att()
    q, k, v, g = make(1, 64, 200, 2, 2, 64, DT[dt], seed=2)
    q = (q.float() * 12).to(DT[dt])
    for scale in (1.0, -0.3, 0.0):
        o = torch.full_like(q, 7.0); l = torch.empty(1, 2, 64, device="cuda")
        out, lse = A.cross_attention(q, k, v, scale=scale, return_lse=True, out=o, lse=l)
        assert out is o and lse is l
        want = R.attend(q, k, v, scale=scale)
        check(out, want[0], bounds(q, k, v, None, None, scale), "out", DT[dt])


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("Tq,Tk", [(6, 50), (90, 600)])
def test_lengths_outside_the_range_and_garbage_behind_them(Tq, Tk, dt):
    """Lengths below 0 and above the time axis count as its ends; rows of q and dout behind a length (NaN, inf, the type's lowest value) leave no trace."""
    A = _att()
    t = DT[dt]
    q, k, v, g = make(4, Tq, Tk, 4, 2, 32, t, seed=Tk)
    ql, kl = lens(Tq + 9, 3, -2, 5), lens(Tk, Tk + 100, 7, -1)
    clean = [x.clone() for x in (q, k, v, g)]
    for x, n in ((q, ql), (g, ql), (k, kl), (v, kl)):
        for i, junk in enumerate((math.nan, math.inf, -math.inf, torch.finfo(t).min)):
            x[i, max(0, int(n[i])):] = junk
    res = []
    for a, b, c, d in ((q, k, v, g), clean):
        o, l = A.cross_attention(a, b, c, k_lens=kl, q_lens=ql, return_lse=True)
        res.append((o, l) + A.cross_attention_grad(d, a, b, c, o, l, k_lens=kl, q_lens=ql))
    assert all(torch.equal(x, y) and not torch.isnan(x).any() for x, y in zip(*res))
    o, l, dq, dk, dv = res[0]
    for i, (m, n) in enumerate(((Tq, Tk), (3, Tk), (0, 7), (5, 0))):
        assert (o[i, m:] == 0).all() and torch.isneginf(l[i, :, m:]).all() and (dq[i, m:] == 0).all() and (dk[i, n:] == 0).all() and (dv[i, n:] == 0).all()
    assert (dk[2] == 0).all() and (o[3] == 0).all() and (dq[3] == 0).all()


def test_scores_of_any_size():
    """fp32 scores around +-1e32 and -1e36 on every key: the softmax is that of their differences (0 or not of this world)."""
    A = _att()
    k = torch.ones(1, 40, 1, 8, device="cuda"); v = torch.randn(1, 40, 1, 8, device="cuda")
    for Tq in (1, 50):
        for s in (1e32, -1e32, -1e36):
            q = torch.full((1, Tq, 1, 8), s / 8, device="cuda")
            out, lse = A.cross_attention(q, k, v, scale=1.0, return_lse=True)
            assert torch.allclose(out, v.mean(1, keepdim=True).expand_as(out), rtol=0, atol=40 * 2.0 ** -23) and torch.isfinite(lse).all()
            for d in A.cross_attention_grad(torch.ones_like(out), q, k, v, out, lse, scale=1.0):
                assert not torch.isnan(d).any()
    q = torch.zeros(1, 70, 1, 16, device="cuda", dtype=torch.float16); q[..., 0] = 60000.0      # fp16: scores to 6e8, one key ahead of the others
    k = torch.zeros(1, 90, 1, 16, device="cuda", dtype=torch.float16); k[0, :, 0, 0] = torch.linspace(0, 10000, 90).half()
    v = torch.randn(1, 90, 1, 16, device="cuda").half()
    for n in (1, 70):
        assert torch.equal(A.cross_attention(q[:, :n], k, v, scale=1.0), v[:, 89:].expand(1, n, 1, 16))


def test_scores_that_are_not_finite():
    """An infinite key: rows whose score is +inf are NaN as softmax has it; a row that meets only -inf has nothing to attend to."""
    A = _att()
    q, k, v, _ = make(1, 40, 3, 1, 1, 16, torch.float32, seed=3)
    q.zero_(); q[..., 0] = 1.0; q[0, 7, 0, 0] = -1.0
    k.zero_(); k[..., 0] = -math.inf
    out, lse = A.cross_attention(q, k, v, return_lse=True)
    keep = torch.arange(40, device="cuda") != 7
    assert (out[0, keep] == 0).all() and torch.isneginf(lse[0, 0, keep]).all() and torch.isnan(out[0, 7]).all()


@pytest.mark.parametrize("rows", [1, 40])
def test_graph_stream_and_reuse(rows):
    """Captured on a side stream, replayed with eager work between, twice in one graph: every replay equals the eager result on the inputs of the moment."""
    A = _att()
    q, k, v, g = make(2, rows, 700, 4, 2, 64, torch.bfloat16, seed=6)
    kl = lens(700, 450)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        A.cross_attention(q, k, v, k_lens=kl)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=st):
        o1, l1 = A.cross_attention(q, k, v, k_lens=kl, return_lse=True)
        d1 = A.cross_attention_grad(g, q, k, v, o1, l1, k_lens=kl)
        o2 = A.cross_attention(q, v, k, k_lens=kl)
    for i in range(4):
        q.copy_(make(2, rows, 700, 4, 2, 64, torch.bfloat16, seed=20 + i)[0]); kl.copy_(lens(700 - 100 * i, 5 + i))
        gr.replay()
        eo, el = A.cross_attention(q, k, v, k_lens=kl, return_lse=True)
        ed = A.cross_attention_grad(g, q, k, v, eo, el, k_lens=kl)
        torch.cuda.synchronize()
        assert torch.equal(o1, eo) and torch.equal(l1, el) and all(torch.equal(x, y) for x, y in zip(d1, ed))
        assert torch.equal(o2, A.cross_attention(q, v, k, k_lens=kl))


def test_empty_sizes():
    A = _att()
    q, k, v, g = make(2, 3, 5, 2, 1, 16, torch.float32)
    out, lse = A.cross_attention(q, k[:, :0], v[:, :0], return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()
    dq, dk, dv = A.cross_attention_grad(g, q, k[:, :0], v[:, :0], out, lse)
    assert (dq == 0).all() and dk.numel() == 0
    assert A.cross_attention(q[:, :0], k, v).shape == (2, 0, 2, 16) and A.cross_attention(q[:0], k[:0], v[:0]).numel() == 0
    o = torch.empty(2, 0, 2, 16, device="cuda"); l = torch.empty(2, 2, 0, device="cuda")
    dq, dk, dv = A.cross_attention_grad(o, q[:, :0], k, v, o, l)
    assert (dk == 0).all() and (dv == 0).all()


# ------------------------------------------------------------------------------------------------ the 8-bit cache
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("T,H,D,kl", [(1, 1, 8, None), (64, 2, 64, (64, 63)), (189, 3, 40, (189, 0)), (300, 2, 128, (65, 300))])
def test_cache_holds_the_defined_values(dt, T, H, D, kl):
    A = _att()
    t = DT[dt]
    B = 1 if kl is None else 2
    _, k, v, _ = make(B, 1, T, H, H, D, t, seed=T)
    k = (k.float() * torch.logspace(-4, 3, T, device="cuda")[None, :, None, None]).to(t)
    v[:, : T // 2] *= 0.0                                          # blocks of zeros
    kl_ = None if kl is None else lens(*kl)
    c = A.EncoderCache8(B, T, H, D)
    c.store(k, v, kl_)
    for x, y, s in ((k, c.k8, c.k_scale), (v, c.v8, c.v_scale)):
        w, ws = R.quantise(x, kl)
        assert torch.equal(s.double(), ws) and torch.equal(y.float().double(), w)
    assert c.lens.tolist() == ([T] if kl is None else list(kl))


def test_cache_values_that_are_not_finite_tiny_or_at_the_border():
    A = _att()
    _, k, v, _ = make(1, 1, 64, 2, 2, 16, torch.float32, seed=1)
    k[0, 3, 0, 1] = math.inf; k[0, 4, 0, 2] = -math.inf; k[0, 5, 0, 3] = math.nan
    k[0, :, 1] = 448.0 * 2.0 ** -20; k[0, 0, 1, 0] = 448.5 * 2.0 ** -20                        # just past the border: the next scale
    v[0, :, 0] *= 2.0 ** -140; v[0, :, 1] = torch.linspace(-448, 448, 64 * 16, device="cuda").view(64, 16)
    c = A.EncoderCache8(1, 64, 2, 16)
    c.store(k, v)
    for x, y, s in ((k, c.k8, c.k_scale), (v, c.v8, c.v_scale)):
        w, ws = R.quantise(x)
        got = y.float().double()
        assert torch.equal(s.double(), ws) and torch.equal(torch.isnan(got), torch.isnan(w)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(w))
    assert c.k_scale[0, 1, 0].item() == 2.0 ** -19 and c.v_scale[0, 0, 0].item() == 2.0 ** -118


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("B,Tq,Tk,Hq,H,D,kl", [(1, 1, 1, 1, 1, 8, None), (1, 1, 189, 8, 8, 64, None), (3, 1, 700, 8, 2, 128, (700, 0, 65)),
                                               (2, 5, 1140, 8, 2, 72, (1140, 1089)), (2, 9, 130, 8, 2, 40, (130, 2)), (1, 1, 5000, 4, 4, 96, None), (2, 40, 200, 2, 2, 16, (199, 64))])
def test_cache_attention(B, Tq, Tk, Hq, H, D, kl, dt):
    A = _att()
    q, k, v, _ = make(B, Tq, Tk, Hq, H, D, DT[dt], seed=Tk + 1)
    k = (k.float() * torch.linspace(0.2, 2, Tk, device="cuda")[None, :, None, None]).to(DT[dt])       # every block its own scale
    v = (v.float() * torch.logspace(2, -2, Tk, device="cuda")[None, :, None, None]).to(DT[dt])
    kl = None if kl is None else lens(*kl)
    c = A.EncoderCache8(B, Tk, H, D)
    c.store(k, v, kl)
    wide = lambda y, s: (y.float().double() * s.double().repeat_interleave(64, 2)[..., None])[:, :, :Tk].transpose(1, 2)  # noqa: E731
    kd, vd = wide(c.k8, c.k_scale), wide(c.v8, c.v_scale)
    want = R.attend(q, kd, vd, kl)
    check(c.attend(q), want[0], bounds(q, kd, vd, kl, None, None), "out", DT[dt])


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("Tk", [256, 1100])
def test_cache_blocks_of_very_different_size(dt, Tk):
    """V's blocks from the largest numbers to the smallest a result can show; columns that only small blocks reach; keys that pick one block."""
    A = _att()
    q, k, v, _ = make(1, 3, Tk, 2, 1, 32, torch.float32, seed=Tk)
    size = (6e4, 1e-7, 1.0, 1e-12) if dt == "f16" else (1e25, 1e-25, 1.0, 1e12)
    blocks = torch.arange(Tk, device="cuda") // 64 % 4
    v = torch.sign(v) * torch.tensor(size, device="cuda")[blocks][None, :, None, None]
    v[:, :, :, 8:16] *= (blocks != 0)[None, :, None, None]
    v[:, :, :, 16:24] *= (blocks == 1)[None, :, None, None]
    k[:, :, :, 0] = torch.tensor((-40.0, 0.0, 40.0, 0.0), device="cuda")[blocks][None, :, None]
    q = q.to(DT[dt])
    q[:, 0, :, 0] = 4.0; q[:, 1, :, 0] = -4.0; q[:, 2, :, 0] = 0.0                             # block 2 decides; block 0 does; all alike
    c = A.EncoderCache8(1, Tk, 1, 32)
    c.store(k, v)
    wide = lambda y, s: (y.float().double() * s.double().repeat_interleave(64, 2)[..., None])[:, :, :Tk].transpose(1, 2)  # noqa: E731
    kd, vd = wide(c.k8, c.k_scale), wide(c.v8, c.v_scale)
    check(c.attend(q), R.attend(q, kd, vd)[0], bounds(q, kd, vd, None, None, None), "out", DT[dt])


def test_cache_appends_blocks_and_replays():
    """A streaming encoder's chunks, an utterance that ends early, queries of another type than the stored one, and a captured step over later stores."""
    A = _att()
    q, k, v, _ = make(2, 1, 300, 4, 2, 64, torch.bfloat16, seed=5)
    c, d = A.EncoderCache8(2, 300, 2, 64), A.EncoderCache8(2, 300, 2, 64)
    c.store(k[:, :128], v[:, :128], lens(128, 100)); c.store(k[:, 128:], v[:, 128:], lens(172, 0), first=128)
    d.store(k, v, lens(300, 100))
    assert c.lens.tolist() == [300, 100] == d.lens.tolist()
    assert torch.equal(c.k8.view(torch.uint8), d.k8.view(torch.uint8)) and torch.equal(c.v_scale, d.v_scale)
    for t in DT.values():
        assert torch.equal(c.attend(q.to(t)), d.attend(q.to(t)))
    gr = torch.cuda.CUDAGraph()
    c.attend(q); torch.cuda.synchronize()
    with torch.cuda.graph(gr):
        o = c.attend(q)
    for i in range(3):
        _, k2, v2, _ = make(2, 1, 300, 4, 2, 64, torch.bfloat16, seed=50 + i)
        c.store(k2, v2, lens(300 - i, 64 * i)); gr.replay(); d.store(k2, v2, lens(300 - i, 64 * i))
        e = d.attend(q); torch.cuda.synchronize()
        assert torch.equal(o, e)


def test_refusals():
    A = _att()
    q, k, v, g = make(2, 3, 5, 4, 2, 16, torch.float32)
    bad = [lambda: A.cross_attention(q, k.half(), v.half()), lambda: A.cross_attention(q, k, v[:, :4]), lambda: A.cross_attention(q[..., :12], k[..., :12], v[..., :12]),
           lambda: A.cross_attention(q[:, :, :3], k, v), lambda: A.cross_attention(q.double(), k.double(), v.double()), lambda: A.cross_attention(q[0], k, v),
           lambda: A.cross_attention(q, k, v, k_lens=torch.tensor([5, 5])), lambda: A.cross_attention(q, k, v, k_lens=lens(5)),
           lambda: A.cross_attention(q, k, v, out=torch.empty(2, 3, 4, 8, device="cuda")), lambda: A.cross_attention(q.cpu(), k.cpu(), v.cpu()),
           lambda: A.cross_attention_grad(g[:, :2], q, k, v, q, torch.empty(2, 4, 3, device="cuda")), lambda: A.EncoderCache8(1, 10, 2, 200), lambda: A.EncoderCache8(0, 10, 2, 64)]
    c = A.EncoderCache8(2, 100, 2, 16)
    kk = torch.zeros(2, 64, 2, 16, device="cuda")
    bad += [lambda: c.store(kk, kk, first=32), lambda: c.store(kk, kk, first=64), lambda: c.store(kk[:1], kk[:1]), lambda: c.attend(q[:, :, :3]), lambda: c.attend(q[:1])]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            print("not refused:", i)
