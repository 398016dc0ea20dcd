"""Gradients of cross attention on the GPU against the float64 formulas, where the operand types' range and the larger calls' kernels come in.

Tolerances: the derivation at the head of test_gpu_attention.py (bounds), which counts relative roundings only -- a ds or p below the operand type's
smallest normal number, or above its largest, has no place in it."""
import math

import pytest
import torch

from tests import _attn_ref as R
from tests.test_gpu_attention import DT, bounds, check, lens, make

pytestmark = pytest.mark.gpu


def _att():
    from aesrc2020_amd import attention
    return attention


def run_and_check(q, k, v, g, kl=None, ql=None, scale=None):
    A, dt = _att(), q.dtype
    out, lse = A.cross_attention(q, k, v, k_lens=kl, q_lens=ql, scale=scale, return_lse=True)
    got = A.cross_attention_grad(g, q, k, v, out, lse, k_lens=kl, q_lens=ql, scale=scale)
    want, bd = R.attend(q, k, v, kl, ql, scale, dout=g), bounds(q, k, v, kl, ql, scale, g)
    check(out, want[0], bd[0], "out", dt)
    for x, w, e, n in zip(got, want[2:], bd[1:], ("dq", "dk", "dv")):
        check(x, w, e, n, dt)
    return got


#         B, Tq,   Tk, Hq, Hkv, D: one launch up to 64 keys; delta from the probabilities up to 256; above; slices of either axis
SIZES = [(2, 70, 39, 4, 2, 64), (1, 150, 64, 2, 2, 128), (2, 90, 200, 4, 2, 128), (1, 130, 1100, 4, 2, 64), (1, 700, 4096, 1, 1, 128), (1, 40, 16000, 1, 1, 32)]


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("size", [1e-5, 1e-4, 1e-2, 2e3])
@pytest.mark.parametrize("shape", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_gradients_for_dout_of_any_size(shape, size, dt):
    """dout of a mean over a batch (1e-4 and less), and large ones: dq, dk and dv are as near as their own rounding lets them be."""
    B, Tq, Tk, Hq, Hkv, D = shape
    q, k, v, g = make(B, Tq, Tk, Hq, Hkv, D, DT[dt], seed=Tk)
    run_and_check(q, k, v, (g.float() * size).to(DT[dt]))


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("shape", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_gradients_of_rows_of_very_different_dout(shape, dt):
    """Tokens whose dout grows along the axis (every tile's larger than the last one's), shrinks, and is zero in between; a key that few rows see."""
    B, Tq, Tk, Hq, Hkv, D = shape
    q, k, v, g = make(B, Tq, Tk, Hq, Hkv, D, DT[dt], seed=Tk + 1)
    e = torch.linspace(-4, 2, Tq, device="cuda")
    for f in (10.0 ** e, 10.0 ** e.flip(0), torch.where(torch.arange(Tq, device="cuda") % 3 == 0, 0.0, 1.0) * 10.0 ** e):
        run_and_check(q, k, v, (g.float() * f[None, :, None, None]).to(DT[dt]))


@pytest.mark.parametrize("dt", DT)
def test_a_power_of_two_on_dout_is_one_on_the_gradients(dt):
    """Where no result leaves the type's normal numbers, bit for bit.  (fp16: upwards only -- a dout below 2^-12 has bits that 2^-2 of it has not.)"""
    A = _att()
    for shape in SIZES[:4]:
        q, k, v, g = make(*shape, DT[dt], seed=3)
        out, lse = A.cross_attention(q, k, v, return_lse=True)
        base = A.cross_attention_grad(g, q, k, v, out, lse)
        for e in (6, 3) if dt == "f16" else (20, -20):
            for x, y in zip(base, A.cross_attention_grad((g.float() * 2.0 ** e).to(DT[dt]), q, k, v, out, lse)):
                normal = (x.abs() >= torch.finfo(DT[dt]).tiny * 2.0 ** max(0, -e)) & (y.float().abs() >= torch.finfo(DT[dt]).tiny)
                assert torch.isfinite(y).all() and torch.equal((x.float() * 2.0 ** e)[normal], y.float()[normal]), (shape, e)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("scale", [0.4, -0.3, 0.0])
@pytest.mark.parametrize("shape", [(2, 70, 39, 4, 2, 64), (1, 130, 200, 4, 2, 128), (2, 90, 300, 2, 1, 40)], ids=lambda s: "x".join(map(str, s)))
def test_given_scales(shape, scale, dt):
    """Negative ones and 0 (every key alike, nothing flows to q and k) too."""
    B, Tq, Tk, Hq, Hkv, D = shape
    q, k, v, g = make(B, Tq, Tk, Hq, Hkv, D, DT[dt], seed=Tk + 2)
    kl = lens(*(Tk - 5 * i for i in range(B)))
    _, dq, dk, _ = (None,) + run_and_check(q, k, v, g, kl, None, scale)
    if scale == 0.0:
        assert (dq == 0).all() and (dk == 0).all()


#         B,  Tq,  Tk, Hq, Hkv, D: 512 blocks of 128 rows, of 128 keys and more: four waves to a block
LARGE = [(16, 500, 77, 8, 8, 64), (16, 500, 201, 16, 8, 40), (16, 450, 301, 8, 8, 128), (32, 37, 300, 8, 8, 64), (43, 130, 390, 8, 4, 96), (9, 1000, 150, 8, 8, 128), (22, 1, 8100, 2, 1, 32),
         (70, 300, 33, 8, 4, 72)]


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("shape", LARGE, ids=lambda s: "x".join(map(str, s)))
def test_blocks_of_four_waves(shape, dt):
    """The kernels that large calls take, with ragged lengths, an utterance without frames and one without rows."""
    B, Tq, Tk, Hq, Hkv, D = shape
    q, k, v, g = make(B, Tq, Tk, Hq, Hkv, D, DT[dt], seed=B)
    i = torch.arange(B, device="cuda")
    kl, ql = (Tk - i * Tk // (2 * B)).int(), (Tq - i * Tq // (2 * B)).int()
    kl[1] = 0; kl[2] = 1; ql[3] = 0
    for b in range(B):
        k[b, int(kl[b]):] = math.nan; v[b, int(kl[b]):] = math.nan
    dead = torch.arange(Tk, device="cuda")[None, :] >= kl[:, None]
    A = _att()
    out, lse = A.cross_attention(q, k, v, k_lens=kl, q_lens=ql, return_lse=True)
    got = A.cross_attention_grad(g, q, k, v, out, lse, k_lens=kl, q_lens=ql)
    for x in (k, v):
        x.masked_fill_(dead[:, :, None, None], 0.0)
    want, bd = R.attend(q, k, v, kl, ql, dout=g), bounds(q, k, v, kl, ql, None, g)
    check(out, want[0], bd[0], "out", DT[dt])
    for x, w, e, n in zip(got, want[2:], bd[1:], ("dq", "dk", "dv")):
        check(x, w, e, n, DT[dt])
    again = A.cross_attention_grad(g, q, k, v, out, lse, k_lens=kl, q_lens=ql)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
