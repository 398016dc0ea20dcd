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
