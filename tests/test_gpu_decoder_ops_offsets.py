"""Tensors of more than 2^31 elements: every offset of the decoder operators past 32 bits.  References in float64, in pieces."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


@pytest.fixture(autouse=True)
def _free():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("Tq", [2, 70])
def test_attention_over_sixteen_million_frames(Tq):
    """2^24 + 100 frames of 128 in fp16; a few frames (first, middle, last) that stand out, so that a wrong offset is a wrong result."""
    from aesrc2020_amd.attention import EncoderCache8, cross_attention, cross_attention_grad
    T, D, step = (1 << 24) + 100, 128, 1 << 20
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(1, Tq, 1, D, generator=g, device="cuda").half()
    k, v = (torch.empty(1, T, 1, D, device="cuda", dtype=torch.float16) for _ in range(2))
    for x, f in ((k, 0.2), (v, 0.25)):
        for i in range(0, T, step):
            x[:, i:i + step] = (torch.randn(1, min(step, T - i), 1, D, generator=g, device="cuda") * f).half()
    at = [0, 1, T // 2, T - 200, T - 2, T - 1]
    for j, i in enumerate(at):
        k[0, i, 0] = (1.2 * q[0, j % Tq, 0].float()).half()
        v[0, i, 0] = 1.0 + j
    do = (torch.randn(1, Tq, 1, D, generator=g, device="cuda") * 0.1).half()
    qd, dd = q[0, :, 0].double(), do[0, :, 0].double()
    scale = D ** -0.5

    def sums(p, x):                                                # p @ x, the long axis in pieces (one float64 product over it takes a tenth of a second)
        n = p.shape[1]
        if n % 4096:
            return p @ x
        return (p.view(Tq, -1, 4096).transpose(0, 1).contiguous() @ x.reshape(-1, 4096, D)).sum(0)

    def pieces(keys, values):
        for i in range(0, T, step):
            yield i, scale * (qd @ keys(i, i + step).T), values(i, i + step)

    def reference(keys, values):
        m = torch.full((Tq, 1), -math.inf, dtype=torch.float64, device="cuda")
        for _, s, _ in pieces(keys, values):
            m = torch.maximum(m, s.amax(1, keepdim=True))
        l, o, w = torch.zeros_like(m), torch.zeros(Tq, D, dtype=torch.float64, device="cuda"), torch.zeros(Tq, D, dtype=torch.float64, device="cuda")
        for _, s, x in pieces(keys, values):
            p = torch.exp(s - m)
            l += p.sum(1, keepdim=True); o += sums(p, x); w += sums(p, x.abs())
        return m + torch.log(l), o / l, w / l

    rows = lambda x: lambda a, b: x[0, a:b, 0].double()  # noqa: E731
    lse, want, size = reference(rows(k), rows(v))
    out, got = cross_attention(q, k, v, return_lse=True)
    # p rounded (u of the sum of p |v|), the result's rounding, the scores' and the sums' fp32 errors
    assert ((out[0, :, 0].double() - want).abs() <= U[q.dtype] * (1.1 * size + want.abs()) + 1e-4 * size).all()
    assert (got[0, 0].double() - lse[:, 0]).abs().max() <= 1e-4
    c = EncoderCache8(1, T, 1, D)
    c.store(k, v)
    held = lambda y, s: lambda a, b: (y[0, 0, a:min(b, T)].float() * s[0, 0, a // 64:-(-min(b, T) // 64)].repeat_interleave(64)[:min(b, T) - a, None]).double()  # noqa: E731
    _, want8, size8 = reference(held(c.k8, c.k_scale), held(c.v8, c.v_scale))
    assert ((c.attend(q)[0, :, 0].double() - want8).abs() <= U[q.dtype] * (1.1 * size8 + want8.abs()) + 1e-4 * size8).all()
    del c
    dq, dk, dv = cross_attention_grad(do, q, k, v, out, got)
    delta = (dd * out[0, :, 0].double()).sum(1, keepdim=True)      # (from the rounded out, as above 256 keys)
    wq, sq = torch.zeros_like(qd), torch.zeros_like(qd)
    for i, s, x in pieces(rows(k), rows(v)):
        p = torch.exp(s - lse)
        dp, ap = dd @ x.T, dd.abs() @ x.abs().T
        ds, ads = p * (dp - delta), p * (ap + delta.abs())
        kk = k[0, i:i + step, 0].double()
        wq += scale * sums(ds, kk); sq += scale * (sums(ds.abs(), kk.abs()) + 1e-3 * sums(ads, kk.abs()))
        e = slice(i, i + step)
        for x_, w_, a_ in ((dk, scale * ds.T @ qd, scale * (ds.abs().T @ qd.abs() + 1e-3 * (ads.T @ qd.abs()))), (dv, p.T @ dd, p.T @ dd.abs())):
            # ds or p rounded (u), fp32 errors of scores and sums (1e-3 of the terms at most), the result's rounding and fp16's smallest step
            assert ((x_[0, e, 0].double() - w_).abs() <= U[q.dtype] * (1.1 * a_ + w_.abs()) + 1e-3 * a_ + 2.0 ** -25).all(), i
    assert ((dq[0, :, 0].double() - wq).abs() <= U[q.dtype] * (1.1 * sq + wq.abs()) + 1e-3 * sq).all()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_vocabulary_loss_of_many_wide_rows(dt):
    """2^21 + 5 rows of 1032 (2.2 G elements) over 70 entries: the last rows' loss and dx, and dkernel, whose sum runs over all of them."""
    from aesrc2020_amd.losses import vocab_crossentropy, vocab_crossentropy_grad
    R, D, V, step = (1 << 21) + 5, 1032, 70, 1 << 17
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.empty(R, D, device="cuda", dtype=dt)
    for i in range(0, R, step):
        x[i:i + step] = torch.randn(min(step, R - i), D, generator=g, device="cuda").to(dt)
    w = (torch.randn(D, V, generator=g, device="cuda") * D ** -0.5).to(dt)
    lab = torch.randint(0, V, (R,), generator=g, device="cuda", dtype=torch.int32)
    dl = torch.rand(R, generator=g, device="cuda") / R
    loss, lse = vocab_crossentropy(x, w, lab, return_lse=True)
    dx, dw, _ = vocab_crossentropy_grad(dl, x, w, lab, lse)
    want, size = torch.zeros(D, V, dtype=torch.float64, device="cuda"), torch.zeros(D, V, dtype=torch.float64, device="cuda")
    for i in range(0, R, step):
        xs, ls, gs = x[i:i + step].double(), lab[i:i + step].long(), dl[i:i + step].double()
        z = xs @ w.double()
        t = torch.logsumexp(z, 1)
        hot = torch.nn.functional.one_hot(ls, V).double()
        dz = gs[:, None] * (torch.softmax(z, 1) - hot)
        want += xs.T @ dz; size += xs.abs().T @ dz.abs()
        if i == 0 or i + 2 * step >= R:
            # fp32 logits and statistics; dz to 11 bits (fp32 22), the result's rounding
            assert ((loss[i:i + step].double() - (t - (z * hot).sum(1))).abs() <= 1e-5).all()
            u = 2.0 ** -11 if dt == torch.bfloat16 else 2.0 ** -18
            wx = dz @ w.double().T
            assert ((dx[i:i + step].double() - wx).abs() <= U[dt] * wx.abs() + u * (dz.abs() @ w.double().abs().T) + 1e-12).all()
    assert ((dw.double() - want).abs() <= U[dt] * want.abs() + (2.0 ** -11 if dt == torch.bfloat16 else 2.0 ** -16) * size).all()


@pytest.mark.parametrize("dt", [torch.float16, torch.float32])
def test_vocabulary_kernel_of_many_elements(dt):
    """A kernel of 65536 x 33000 (2.2 G elements) under 70 rows: loss, dx, and dkernel's first and last rows."""
    from aesrc2020_amd.losses import vocab_crossentropy, vocab_crossentropy_grad
    R, D, V, step = 70, 65536, 33000, 4096
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(R, D, generator=g, device="cuda").to(dt)
    w = torch.empty(D, V, device="cuda", dtype=dt)
    for i in range(0, D, step):
        w[i:i + step] = (torch.randn(step, V, generator=g, device="cuda") * D ** -0.5).to(dt)
    lab = torch.randint(0, V, (R,), generator=g, device="cuda", dtype=torch.int64)
    lab[0] = V - 1
    dl = torch.rand(R, generator=g, device="cuda")
    loss, lse = vocab_crossentropy(x, w, lab, return_lse=True)
    dx, dw, _ = vocab_crossentropy_grad(dl, x, w, lab, lse)
    z = torch.zeros(R, V, dtype=torch.float64, device="cuda")
    for i in range(0, D, step):
        z += x[:, i:i + step].double() @ w[i:i + step].double()
    hot = torch.nn.functional.one_hot(lab, V).double()
    assert ((loss.double() - (torch.logsumexp(z, 1) - (z * hot).sum(1))).abs() <= 1e-4).all()
    dz = dl.double()[:, None] * (torch.softmax(z, 1) - hot)
    u = 2.0 ** -10 if dt == torch.float16 else 2.0 ** -13          # dz's bits; the logits' fp32 error (65536 products) is a relative one of dz
    for i in list(range(0, D, step))[::5] + [D - step]:
        e = slice(i, i + step)
        wx, ww = dz @ w[e].double().T, x[:, e].double().T @ dz
        assert ((dx[:, e].double() - wx).abs() <= U[dt] * wx.abs() + u * (dz.abs() @ w[e].double().abs().T) + 2.0 ** -24).all(), i
        assert ((dw[e].double() - ww).abs() <= U[dt] * ww.abs() + u * (x[:, e].double().abs().T @ dz.abs()) + (2.0 ** -24 if dt == torch.float16 else 0)).all(), i
