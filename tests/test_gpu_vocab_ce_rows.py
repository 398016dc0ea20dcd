"""Vocabulary cross entropy: what one row holds leaves the other rows' results alone, bit for bit.

Sizes: (20, 48, 130) small tiles, operands as they are in fp32 and bf16; (2000, 256, 700) fp32 gradients from packed operands, small tiles; (1100, 640, 4000) all
types on large tiles, fp32 and bf16 gradients from packed operands; (1100, 637, 4001) the same with rows that have to be copied."""
import math

import pytest
import torch

from tests.test_gpu_vocab_ce import DT, make

pytestmark = pytest.mark.gpu
SIZES = [(20, 48, 130), (2000, 256, 700), (1100, 640, 4000), (1100, 637, 4001)]


def run(dl, x, w, lab, b):
    from aesrc2020_amd.losses import vocab_crossentropy, vocab_crossentropy_grad
    loss, lse = vocab_crossentropy(x, w, lab, b, return_lse=True)
    return (loss, lse) + vocab_crossentropy_grad(dl, x, w, lab, lse, b)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("R,D,V", SIZES)
def test_dloss_of_rows_without_a_label_is_not_looked_at(R, D, V, dt):
    """make() leaves every seventh row out, by -1, and one by V."""
    x, w, lab, b, dl = make(R, D, V, DT[dt], seed=R)
    out = (lab < 0) | (lab >= V)
    want = run(torch.where(out, torch.zeros_like(dl), dl), x, w, lab, b)
    assert all(w_.abs().max() > 0 for w_ in want[2:])
    for junk in (1e6, -1e30, math.inf, math.nan):
        for labels in (lab, lab.long()):
            got = run(torch.where(out, torch.full_like(dl, junk), dl), x, w, labels, b)
            assert all(torch.equal(g, w_) for g, w_ in zip(got, want)), junk


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("R,D,V", SIZES)
def test_a_large_row_without_a_label_leaves_no_trace(R, D, V, dt):
    """x of left-out rows up to what the type holds: every result of the others, and the kernel's and the bias's gradients, bit for bit."""
    x, w, lab, b, dl = make(R, D, V, DT[dt], seed=R)
    out = (lab < 0) | (lab >= V)
    want = run(dl, torch.where(out[:, None], torch.zeros_like(x), x), w, lab, b)
    for size in (6e4,) if dt == "f16" else (1e6, 1e12, 1e20, 1e37):
        got = run(dl, torch.where(out[:, None], torch.full_like(x, size) * torch.sign(x), x), w, lab, b)
        for i, (g, w_) in enumerate(zip(got, want)):
            assert torch.equal(g[~out], w_[~out]) if i in (1, 2) else torch.equal(g, w_), (size, i)
        assert (got[2][out] == 0).all()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("R,D,V", SIZES)
def test_a_large_row_leaves_the_other_rows_alone(R, D, V, dt):
    """A labelled row far larger than the others: their loss, log-sum-exp and dx do not change by a bit."""
    x, w, lab, b, dl = make(R, D, V, DT[dt], seed=R)
    others = torch.arange(R, device="cuda") != 2
    want = run(dl, x, w, lab, b)
    for size in (1e4,) if dt == "f16" else (1e4, 1e6, 1e10, 1e20, 1e30):
        y = x.clone(); y[2] *= size
        got = run(dl, y, w, lab, b)
        assert torch.isfinite(got[0]).all() and torch.isfinite(got[2]).all()
        assert all(torch.equal(g[others], w_[others]) for g, w_ in zip(got[:3], want)), size


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("R,D,V", SIZES[1:])
def test_rows_of_many_sizes(R, D, V, dt):
    """Rows of x over eight orders of magnitude (fp16: five), each held to its own.

    The logits of a row: fp32 sums of D products, |dz| <= 2^-24 (D + 4) sum |x W|; packed fp32 operands add 2^-21 sum |x W| and, for elements far below
    their maxima, 2^-37 D max|x_r| max|W| with x_r THIS row.  lse and loss: as derived in test_gpu_vocab_ce.py.  dx: dz's steps (ed there) met by W."""
    from tests.test_gpu_vocab_ce import check, reference
    x, w, lab, b, dl = make(R, D, V, DT[dt], seed=R + 1)
    e = torch.linspace(-3, 2 if dt == "f16" else 5, R, device="cuda")[torch.randperm(R, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")]
    x = (x.float() * 10.0 ** e[:, None]).to(x.dtype)
    got = run(dl, x, w, lab, b)
    for i in range(0, R, 97):                                      # one row at a time: reference() takes maxima over its rows
        s = slice(i, i + 1)
        want, bd = reference(x[s], w, lab[s], b, dl[s])
        check(got[0][s], want[0], bd[0], "loss"); check(got[1][s], want[1], bd[1], "lse")
        check(got[2][s], want[2], bd[2] + 2.0 ** -38 * dl.abs().max().item() * w.double().abs().sum(1), "dx")


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("R,D,V", SIZES)
def test_powers_of_two_at_the_ends_of_the_range(R, D, V, dt):
    """x up to the type's largest numbers beside a kernel near its smallest, and the other way: the logits are the same, and so are loss and lse, bit for bit;
    the gradient that grows is the same times the power, where it stays within the type.  (The one that shrinks sums numbers below 2^-126.  What is below 2^-14 is left out of the inputs: times 2^-110 the rest
    are normal numbers, with all their bits.)"""
    x, w, lab, b, dl = make(R, D, V, DT[dt], seed=R)
    x, w = (torch.where(t.abs() < 2.0 ** -14, torch.zeros_like(t), t) for t in (x, w))
    base = run(dl, x, w, lab, b)
    for e in (110, -110):
        got = run(dl, (x.float() * 2.0 ** e).to(x.dtype), (w.float() * 2.0 ** -e).to(w.dtype), lab, b)
        assert torch.equal(got[0], base[0]) and torch.equal(got[1], base[1]), e
        y, z = (g[3 if e > 0 else 2].double() for g in (base, got))
        y *= 2.0 ** 110
        fits = y.abs() < 2.0 ** 127
        assert fits.any() and torch.equal(z[fits], y[fits]) and torch.isfinite(got[2]).all() and (e > 0 or torch.isfinite(got[3]).all()), e
    assert torch.equal(got[4], base[4]) if b is not None else True


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("R,D,V", SIZES)
def test_no_row_has_a_label(R, D, V, dt):
    x, w, lab, b, dl = make(R, D, V, DT[dt], seed=R)
    got = run(dl, x, w, torch.full_like(lab, V + 3), b)
    assert (got[0] == 0).all() and torch.equal(got[1], run(dl, x, w, lab, b)[1]) and all((g == 0).all() for g in got[2:] if g is not None)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("R,D,V", SIZES[1:3])
def test_left_out_rows_at_the_end_of_the_range(R, D, V, dt):
    x, w, lab, b, dl = make(R, D, V, DT[dt], seed=R)
    out = (lab < 0) | (lab >= V)
    want = run(dl, torch.where(out[:, None], torch.zeros_like(x), x), w, lab, b)
    got = run(dl, torch.where(out[:, None], torch.full_like(x, torch.finfo(x.dtype).max) * torch.sign(x), x), w, lab, b)
    assert all(torch.equal(g, w_) for i, (g, w_) in enumerate(zip(got, want)) if i != 1)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("R,D,V", SIZES)
def test_the_dloss_of_a_row_leaves_the_other_rows_alone(R, D, V, dt):
    """A labelled row's dloss up to 1e30 and down to 1e-30: dx of the others does not change by a bit, its own follows.  (fp16 holds dz under one scale.)"""
    x, w, lab, b, dl = make(R, D, V, DT[dt], seed=R)
    others = torch.arange(R, device="cuda") != 2
    want = run(dl, x, w, lab, b)
    for e in (100, 20, -20, -100):
        d = dl.clone(); d[2] *= 2.0 ** e
        got = run(d, x, w, lab, b)
        assert torch.equal(got[2][others], want[2][others]), e
        y, z = want[2][2].double() * 2.0 ** e, got[2][2].double()
        # (in the type's normal numbers; fp32 sums of what lies below them lose bits)
        assert e < -20 or torch.equal(z, y), e
        assert all(torch.isfinite(t).all() for t in got[2:] if t is not None)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("R,D,V", SIZES[1:])
def test_rows_of_many_dlosses(R, D, V, dt):
    """dloss over twelve orders of magnitude: dx row by row against float64 (each row alone: reference() takes maxima over its rows), dkernel and dbias as a
    whole, dkernel's packed x adding 2^-37 max |x dloss| for each row's softmax - onehot."""
    from tests.test_gpu_vocab_ce import check, reference
    x, w, lab, b, dl = make(R, D, V, DT[dt], seed=R + 2)
    g = torch.Generator(device="cuda").manual_seed(1)
    dl = dl * 10.0 ** torch.linspace(-6, 6, R, device="cuda")[torch.randperm(R, generator=g, device="cuda")]
    got = run(dl, x, w, lab, b)
    for i in range(0, R, 97):
        s = slice(i, i + 1)
        want, bd = reference(x[s], w, lab[s], b, dl[s])
        check(got[2][s], want[2], bd[2], "dx")
    want, bd = reference(x, w, lab, b, dl)
    check(got[3], want[3], bd[3] + 2.0 ** -37 * (x.double().abs().amax(1) * dl.double().abs()).max(), "dkernel")
    if b is not None:
        check(got[4], want[4], bd[4], "dbias")
