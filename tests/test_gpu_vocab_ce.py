"""Softmax cross entropy over a vocabulary on the GPU against the float64 definition.

Tolerances.  u = half a step of the type (finfo.eps / 2), f = 2^-24.
  z: products of the 16-bit types are exact and summed in fp32: |dz| <= f (D + 4) sum |x W| (sequential sums at worst); fp32 operands are two fp16
  planes under a tensor-wide scale: relative 2^-21 more of |x||W| (hi + lo: 2^-23 each side; lo lo dropped: 2^-22), and 2^-38 of the tensors' maxima
  for elements far below them.  lse: the same error plus f (V/8 + |lse| + 32).  loss: both.
  dz = g (p - onehot): relative error (ez + else) of p, rounded to the operand type (u; fp32: 2^-22), at least 2^-39 of the largest |g| in absolute terms
  (fp16 operands' smallest step under the scale 2^14).  dx, dW, db: those times the other operand's magnitudes, sums f n, the result's rounding u."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def make(R, D, V, dt, bias=True, seed=0, amp=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(R, D, generator=g, device="cuda").to(dt)
    w = (torch.randn(D, V, generator=g, device="cuda") * (amp / math.sqrt(D))).to(dt)
    b = (torch.randn(V, generator=g, device="cuda") * 0.5).to(dt) if bias else None
    lab = torch.randint(0, V, (R,), generator=g, device="cuda", dtype=torch.int32)
    lab[:: 7] = -1
    if R > 3:
        lab[3] = V                                                 # outside as well
    if R > 1:
        lab[1] = V - 1
    dl = (torch.rand(R, generator=g, device="cuda") - 0.3) / R
    return x, w, lab, b, dl


def reference(x, w, lab, b, dl):
    """float64 values and elementwise bounds: (loss, lse, dx, dw, db), (bounds of the same)."""
    t = x.dtype
    f, u = 2.0 ** -24, torch.finfo(t).eps / 2
    R, D = x.shape
    V = w.shape[1]
    x, w, dl = x.double(), w.double(), dl.double()
    z, za = x @ w, x.abs() @ w.abs()
    if b is not None:
        z = z + b.double(); za = za + b.double().abs()
    ez = f * (D + 4) * za
    if t == torch.float32:
        ez = ez + 2.0 ** -21 * za + 2.0 ** -37 * D * x.abs().max() * w.abs().max()
    lse = torch.logsumexp(z, 1)
    p = torch.softmax(z, 1)
    es = (p * ez).sum(1) + ez.amax(1) * 0 + f * (V / 8 + 2 * lse.abs() + 4 * z.abs().amax(1) + 32)
    lab = lab.long()
    has = (lab >= 0) & (lab < V)
    at = torch.where(has, lab, torch.zeros_like(lab))[:, None]
    loss = torch.where(has, lse - z.gather(1, at)[:, 0], torch.zeros_like(lse))
    el = torch.where(has, es + ez.gather(1, at)[:, 0] + f * (lse.abs() + z.gather(1, at)[:, 0].abs()), torch.zeros_like(es))
    g = torch.where(has, dl, torch.zeros_like(dl))[:, None]
    hot = torch.zeros_like(z).scatter_(1, at, 1.0)
    dz = g * (p - hot)
    rel = ez + es[:, None] + f * (4 * (z - lse[:, None]).abs() + 8)
    ud = 2.0 ** -21 if t == torch.float32 else u
    ed = g.abs() * p * rel * (1 + rel) + ud * dz.abs() * (1 + rel) + 2.0 ** -38 * g.abs().max() + f * 4 * dz.abs()
    extra = 2.0 ** -21 if t == torch.float32 else 0.0
    dx, edx = dz @ w.T, ed @ w.abs().T + (f * (V + 64) + extra) * (dz.abs() @ w.abs().T) + (2.0 ** -37 * w.abs().max() * dz.abs().sum(1, keepdim=True) if extra else 0.0)
    dw, edw = x.T @ dz, x.abs().T @ ed + (f * (R + 64) + extra) * (x.abs().T @ dz.abs()) + (2.0 ** -37 * x.abs().max() * dz.abs().sum(0, keepdim=True) if extra else 0.0)
    db, edb = dz.sum(0), ed.sum(0) + f * (R + 8) * dz.abs().sum(0)
    tiny = 2.0 ** -25 if t == torch.float16 else 0.0
    return (loss, lse, dx, dw, db), (el, es, edx + u * dx.abs() + tiny, edw + u * dw.abs() + tiny, edb + u * db.abs() + tiny)


def check(got, want, bound, what):
    assert torch.isfinite(got).all(), what
    r = ((got.double() - want).abs() / (1.05 * bound + 1e-300))
    assert r.max().item() <= 1.0, (what, r.max().item(), (got.double() - want).abs().max().item())


SHAPES = [(1, 1, 1), (1, 256, 1000), (5, 40, 11), (33, 32, 32), (64, 96, 257), (130, 131, 300), (300, 256, 1000), (77, 512, 4099), (700, 64, 5003), (2, 1024, 20000), (2600, 264, 1000), (40, 72, 30001), (4000, 36, 12), (65, 30, 999)]


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("R,D,V", SHAPES)
def test_loss_and_gradients(R, D, V, dt):
    from aesrc2020_amd.losses import vocab_crossentropy, vocab_crossentropy_grad
    x, w, lab, b, dl = make(R, D, V, DT[dt], bias=V % 2 == 0 or V < 12, seed=R + V)
    want, bd = reference(x, w, lab, b, dl)
    loss, lse = vocab_crossentropy(x, w, lab, b, return_lse=True)
    check(loss, want[0], bd[0], "loss"); check(lse, want[1], bd[1], "lse")
    assert torch.equal(vocab_crossentropy(x, w, lab.long(), b), loss)
    got = vocab_crossentropy_grad(dl, x, w, lab, lse, b)
    names = ("dx", "dkernel", "dbias")
    for g, wv, e, n in zip(got, want[2:], bd[2:], names):
        if g is not None:
            check(g, wv, e, n)
    again = vocab_crossentropy_grad(dl, x, w, lab, lse, b)
    assert all(g is None or torch.equal(g, h) for g, h in zip(got, again))
    only = vocab_crossentropy_grad(dl, x, w, lab, lse, b, need_dx=False)
    assert only[0] is None and torch.equal(only[1], got[1])


@pytest.mark.parametrize("dt", DT)
def test_several_pieces_of_the_vocabulary(dt):
    """Enough rows that a piece is a part of the vocabulary, and the last one is short and odd."""
    from aesrc2020_amd.losses import vocab_crossentropy, vocab_crossentropy_grad
    R, D, V = 8192, 64, 20011 if dt != "f32" else 9003
    x, w, lab, b, dl = make(R, D, V, DT[dt], seed=1)
    want, bd = reference(x, w, lab, b, dl)
    loss, lse = vocab_crossentropy(x, w, lab, b, return_lse=True)
    check(loss, want[0], bd[0], "loss")
    for g, wv, e, n in zip(vocab_crossentropy_grad(dl, x, w, lab, lse, b), want[2:], bd[2:], ("dx", "dkernel", "dbias")):
        check(g, wv, e, n)


@pytest.mark.parametrize("dt", DT)
def test_gradients_against_differences(dt):
    from aesrc2020_amd.losses import vocab_crossentropy, vocab_crossentropy_grad
    x, w, lab, b, dl = make(20, 48, 130, DT[dt], seed=3)
    _, lse = vocab_crossentropy(x, w, lab, b, return_lse=True)
    grads = vocab_crossentropy_grad(dl, x, w, lab, lse, b)
    _, bd = reference(x, w, lab, b, dl)
    gen = torch.Generator(device="cuda").manual_seed(5)
    for i, (t, d) in enumerate(zip((x, w, b), grads)):
        v = torch.randn(t.shape, generator=gen, device="cuda", dtype=torch.float64)
        f = []
        for s in (1, -1):
            a = [y.double() + (s * 1e-5 * v if j == i else 0) for j, y in enumerate((x, w, b))]
            f.append((reference(a[0], a[1], lab, a[2], dl)[0][0] * dl.double()).sum())
        num, ana = ((f[0] - f[1]) / 2e-5).item(), (d.double() * v).sum().item()
        assert abs(num - ana) <= (v.abs() * 1.05 * bd[2 + i]).sum().item() + 1e-8, (i, num, ana)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("R,D,V", [(20, 48, 130), (1100, 640, 4000)])
@pytest.mark.parametrize("e", [100, -60])
def test_gradients_follow_the_size_of_dloss(e, R, D, V, dt):
    """A power of two on dloss is one on the gradients, whatever held dz in between (tiny probabilities may come out as zeros: a quarter of a rounding)."""
    from aesrc2020_amd.losses import vocab_crossentropy, vocab_crossentropy_grad
    x, w, lab, b, dl = make(R, D, V, DT[dt], seed=8)
    _, lse = vocab_crossentropy(x, w, lab, b, return_lse=True)
    for g, h in zip(vocab_crossentropy_grad(dl, x, w, lab, lse, b), vocab_crossentropy_grad(dl * 2.0 ** e, x, w, lab, lse, b)):
        g, h = g.double(), h.double() * 2.0 ** -e
        assert torch.isfinite(h).all() and ((g - h).abs() <= torch.finfo(DT[dt]).eps * g.abs() + 2.0 ** -40 * g.abs().max()).all()


@pytest.mark.parametrize("dt", DT)
def test_strides_scales_and_wide_ranges(dt):
    """Strided and unaligned rows and kernels; tensors far from 1 in size; upstream gradients of one row a million times another's."""
    from aesrc2020_amd.losses import vocab_crossentropy, vocab_crossentropy_grad
    t = DT[dt]
    x, w, lab, b, dl = make(50, 64, 320, t, seed=8)
    base = vocab_crossentropy(x, w, lab, b, return_lse=True)
    wide = torch.zeros(50, 72, device="cuda", dtype=t); wide[:, :64] = x
    kw = torch.zeros(64, 328, device="cuda", dtype=t); kw[:, :320] = w
    raw = torch.zeros(64 * 320 + 1, device="cuda", dtype=t); raw[1:] = w.flatten()
    for xx, ww in ((wide[:, :64], w), (x, kw[:, :320]), (x, raw[1:].view(64, 320)), (x.t().contiguous().t(), w.t().contiguous().t())):
        got = vocab_crossentropy(xx, ww, lab, b, return_lse=True)
        assert torch.equal(got[0], base[0]) and torch.equal(got[1], base[1])
        for p, q in zip(vocab_crossentropy_grad(dl, xx, ww, lab, got[1], b), vocab_crossentropy_grad(dl, x, w, lab, base[1], b)):
            assert torch.equal(p, q)
    for sx, sw in ((2.0 ** 10, 2.0 ** -10), (2.0 ** -8, 2.0 ** 8)):
        x2, w2 = (x.float() * sx).to(t), (w.float() * sw).to(t)
        dl2 = dl * torch.logspace(-6, 0, 50, device="cuda")
        want, bd = reference(x2, w2, lab, b, dl2)
        loss, lse = vocab_crossentropy(x2, w2, lab, b, return_lse=True)
        check(loss, want[0], bd[0], "loss")
        for g, wv, e, n in zip(vocab_crossentropy_grad(dl2, x2, w2, lab, lse, b), want[2:], bd[2:], ("dx", "dkernel", "dbias")):
            check(g, wv, e, n)


def test_large_logits_no_labels_and_zero_gradients():
    from aesrc2020_amd.losses import vocab_crossentropy, vocab_crossentropy_grad
    x, w, lab, b, dl = make(40, 64, 200, torch.float32, seed=2, amp=300.0)
    want, bd = reference(x, w, lab, b, dl)
    loss, lse = vocab_crossentropy(x, w, lab, b, return_lse=True)
    check(loss, want[0], bd[0], "loss")
    for big in (1e9, 1e13):                                        # logits whose rounding is whole units: one-hot, finite, the sum rules hold
        hx = torch.zeros(3, 64, device="cuda"); hx[:, 0] = big
        hw = torch.zeros(64, 200, device="cuda"); hw[0] = torch.linspace(0, 1, 200, device="cuda")
        hl = torch.tensor([199, 5, 0], dtype=torch.int32, device="cuda")
        l2, s2 = vocab_crossentropy(hx, hw, hl, return_lse=True)
        gx, gw, _ = vocab_crossentropy_grad(torch.ones(3, device="cuda"), hx, hw, hl, s2)
        assert torch.allclose(l2.double(), big * (1 - hw[0, hl.long()].double()), rtol=2.0 ** -21, atol=0) and torch.isfinite(gx).all() and torch.isfinite(gw).all()
        p = gw[0].double() / big                                   # sum over the rows of softmax - onehot: the last entry, minus the labels
        want = torch.zeros(200, device="cuda", dtype=torch.float64); want[199] = 2.0; want[5] = want[0] = -1.0
        assert torch.allclose(p, want, rtol=0, atol=1e-5)
    none = torch.full_like(lab, -1)
    assert (vocab_crossentropy(x, w, none, b) == 0).all()
    for d, lb in ((dl, none), (torch.zeros_like(dl), lab)):
        assert all((g == 0).all() for g in vocab_crossentropy_grad(d, x, w, lb, lse, b))
    x[5, 3] = math.nan                                             # one bad row is one bad loss
    bad = vocab_crossentropy(x, w, lab, b)
    ok = torch.ones(40, dtype=torch.bool, device="cuda"); ok[5] = False
    assert torch.equal(bad[ok], loss[ok]) and (torch.isnan(bad[5]) or lab[5] < 0)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("R,D,V", [(40, 72, 202), (40, 50, 201), (40, 64, 192), (300, 136, 20010)])
def test_a_bad_row_stays_alone(R, D, V, dt):
    """NaN in one row of x (its neighbours end inside a contraction step) and in one column of the kernel: only what reads them is NaN; rows that are
    4-byte but not 16-byte aligned."""
    from aesrc2020_amd.losses import vocab_crossentropy, vocab_crossentropy_grad
    t = DT[dt]
    x, w, lab, b, dl = make(R, D, V, t, seed=D)
    loss, lse = vocab_crossentropy(x, w, lab, b, return_lse=True)
    step = 4 // t.itemsize
    raw = torch.zeros(x.numel() + step, device="cuda", dtype=t); raw[step:] = x.flatten()
    rw = torch.zeros(w.numel() + step, device="cuda", dtype=t); rw[step:] = w.flatten()
    x2, w2 = raw[step:].view(R, D), rw[step:].view(D, V)
    l2, s2 = vocab_crossentropy(x2, w2, lab, b, return_lse=True)
    assert torch.equal(l2, loss) and torch.equal(s2, lse)
    for p, q in zip(vocab_crossentropy_grad(dl, x2, w2, lab, s2, b), vocab_crossentropy_grad(dl, x, w, lab, lse, b)):
        assert torch.equal(p, q)
    y = x.clone(); y[20, 0] = math.nan
    bad = vocab_crossentropy(y, w, lab, b)
    ok = torch.ones(R, dtype=torch.bool, device="cuda"); ok[20] = False
    assert torch.equal(bad[ok], loss[ok]) and torch.isnan(bad[20])
    y = x.clone(); y[20] = 0; y[20, 0] = math.inf                  # its row without a label: nothing of it in the gradients but 0 * inf in dkernel's first row
    l3 = lab.clone(); l3[20] = -1
    dx, dw, _ = vocab_crossentropy_grad(dl, y, w, l3, lse, b)
    assert torch.isfinite(dx).all() and torch.isfinite(dw[1:]).all()


@pytest.mark.parametrize("R", [20, 100])
def test_accumulate_empty_and_graph(R):
    from aesrc2020_amd.losses import vocab_crossentropy, vocab_crossentropy_grad
    x, w, lab, b, dl = make(R, 64, 330, torch.float32, seed=4)
    _, lse = vocab_crossentropy(x, w, lab, b, return_lse=True)
    _, dw, db = vocab_crossentropy_grad(dl, x, w, lab, lse, b)
    aw, ab = torch.ones_like(dw), torch.full_like(db, 2.0)
    vocab_crossentropy_grad(dl, x, w, lab, lse, b, dkernel=aw, dbias=ab, accumulate=True)
    assert torch.equal(aw, dw + 1) and torch.equal(ab, db + 2)
    e = vocab_crossentropy_grad(dl[:0], x[:0], w, lab[:0], lse[:0], b)
    assert e[0].shape == (0, 64) and (e[1] == 0).all() and (e[2] == 0).all()
    assert vocab_crossentropy(x[:0], w, lab[:0], b).shape == (0,)
    vocab_crossentropy_grad(dl, x, w, lab, lse, b, dkernel=aw, dbias=ab, accumulate=True)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        l1, s1 = vocab_crossentropy(x, w, lab, b, return_lse=True)
        g1 = vocab_crossentropy_grad(dl, x, w, lab, s1, b)
    for i in range(4):
        x.copy_(make(R, 64, 330, torch.float32, seed=30 + i)[0]); lab.copy_((lab + 17) % 330)
        gr.replay()
        l2, s2 = vocab_crossentropy(x, w, lab, b, return_lse=True)
        g2 = vocab_crossentropy_grad(dl, x, w, lab, s2, b)
        torch.cuda.synchronize()
        assert torch.equal(l1, l2) and all(torch.equal(p, q) for p, q in zip(g1, g2))


def test_refusals():
    from aesrc2020_amd.losses import vocab_crossentropy, vocab_crossentropy_grad
    x, w, lab, b, dl = make(6, 32, 64, torch.bfloat16)
    lse = torch.zeros(6, device="cuda")
    for f in (lambda: vocab_crossentropy(x, w.float(), lab), lambda: vocab_crossentropy(x, w[:16], lab), lambda: vocab_crossentropy(x, w, lab[:5]), lambda: vocab_crossentropy(x, w, lab.float()),
              lambda: vocab_crossentropy(x, w, lab, b[:3]), lambda: vocab_crossentropy(x.cpu(), w.cpu(), lab.cpu()), lambda: vocab_crossentropy(x[0], w, lab),
              lambda: vocab_crossentropy_grad(dl[:5], x, w, lab, lse), lambda: vocab_crossentropy_grad(dl, x, w, lab, lse, accumulate=True),
              lambda: vocab_crossentropy_grad(dl, x, w, lab, lse, dkernel=torch.empty(32, 60, device="cuda", dtype=torch.bfloat16))):
        with pytest.raises(ValueError):
            f()
