"""Vocabulary cross entropy: entries masked through the bias, labels far outside, rows that are certain."""
import math

import pytest
import torch

from tests.test_gpu_vocab_ce import DT, check, make, reference
from tests.test_gpu_vocab_ce_rows import SIZES, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("lowest", [False, True])
@pytest.mark.parametrize("R,D,V", SIZES)
def test_entries_masked_through_the_bias(R, D, V, lowest, dt):
    """-inf, or the type's lowest value, on a third of the entries, whole tiles among them: the result over the others, nothing for the masked."""
    x, w, lab, b, dl = make(R, D, V, DT[dt], seed=V)
    off = torch.zeros(V, dtype=torch.bool, device="cuda")
    off[V // 2:V // 2 + V // 4] = True
    off[::12] = True; off[V - 1] = False; off[0] = True
    lab = torch.where((lab >= 0) & (lab < V) & off[lab.long().clamp(0, V - 1)], torch.full_like(lab, -1), lab)
    masked = torch.where(off, torch.full_like(b, torch.finfo(b.dtype).min if lowest else -math.inf), b)
    keep = (~off).nonzero()[:, 0]
    place = torch.full((V,), -1, dtype=torch.int32, device="cuda"); place[keep] = torch.arange(keep.numel(), dtype=torch.int32, device="cuda")
    mine = torch.where((lab >= 0) & (lab < V), place[lab.long().clamp(0, V - 1)], torch.full_like(lab, -1))
    if lowest and dt == "f16":                                     # (-65504 is a number like any other, far below)
        assert (masked[off] == -65504).all()
    got = run(dl, x, w, lab, masked)
    want, bd = reference(x, w[:, keep], mine, b[keep], dl)
    f = 2.0 ** -24 * V / 8                                         # (sums over V places, not over the kept ones)
    check(got[0], want[0], bd[0] + f, "loss"); check(got[1], want[1], bd[1] + f, "lse")
    check(got[2], want[2], bd[2] + f * (dl.double().abs()[:, None] * w.double().abs().amax(1)), "dx")
    check(got[3][:, keep], want[3], bd[3] + f * want[3].abs(), "dkernel"); check(got[4][keep], want[4], bd[4] + f * want[4].abs(), "dbias")
    assert (got[3][:, off] == 0).all() and (got[4][off] == 0).all()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("R,D,V", SIZES[:3])
def test_labels_beyond_32_bits_leave_their_rows_out(R, D, V, dt):
    x, w, lab, b, dl = make(R, D, V, DT[dt], seed=V)
    far = lab.long()
    for i, l in enumerate((2 ** 32 + 5, -2 ** 32 + 5, 2 ** 62, -2 ** 63, 2 ** 63 - 1, 2 ** 31)):
        far[2 * i] = l
    near = torch.where((far < 0) | (far >= V), torch.full_like(far, -1), far)
    for g, h in zip(run(dl, x, w, far, b), run(dl, x, w, near, b)):
        assert torch.equal(g, h)
    assert (run(dl, x, w, far, b)[0][[0, 2, 4, 6, 8, 10]] == 0).all()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("R,D,V", SIZES)
def test_rows_that_are_certain(R, D, V, dt):
    """x that puts the label's logit 60 above all others: loss 0 (or the sum's rounding), gradients that vanish with 1 - p; beside a row that is certainly wrong."""
    x, w, lab, b, dl = make(R, D, V, DT[dt], seed=V, amp=0.1)
    lab = lab.clamp(0, V - 1)
    x[:, 0] = 1.0; w[0] = -60.0
    w[0, 3] = 0.0
    lab[:] = 3
    lab[-1] = 5
    want, bd = reference(x, w, lab, b, dl)
    got = run(dl, x, w, lab, b)
    for g, t, e, n in zip(got, want, bd, ("loss", "lse")):
        check(g, t, e, n)
    for g, t, e, n in zip(got[2:], want[2:], bd[2:], ("dx", "dkernel", "dbias")):
        check(g, t, e, n)
    assert (got[0][:-1].abs() <= 2.0 ** -15).all() and got[0][-1] > 50
