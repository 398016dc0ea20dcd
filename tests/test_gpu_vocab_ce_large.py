"""Vocabulary cross entropy on the GPU at sizes where grids, tiles and indexes change."""
import math

import pytest
import torch

from tests.test_gpu_vocab_ce import DT, check, make, reference

pytestmark = pytest.mark.gpu


def test_more_tiles_than_one_row_of_a_launch():
    """2^20 rows over 2^18 + 50 entries: 2049 x 8192 tiles, more than 2^32 threads.  A sample of the rows against float64 (bounds: test_gpu_vocab_ce.py)."""
    from aesrc2020_amd.losses import vocab_crossentropy
    R, D, V = 1 << 20, 16, (1 << 18) + 50
    x, w, lab, b, dl = make(R, D, V, torch.bfloat16, seed=1)
    loss, lse = vocab_crossentropy(x, w, lab, b, return_lse=True)
    rows = torch.cat([torch.arange(8), torch.arange(8) + R // 2 - 4, torch.arange(8) + R - 8]).cuda()
    want, bd = reference(x[rows], w, lab[rows], b, dl[rows])
    check(loss[rows], want[0], bd[0], "loss"); check(lse[rows], want[1], bd[1], "lse")
    assert torch.isfinite(lse).all() and (loss[(lab < 0) | (lab >= V)] == 0).all()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("R,D,V", [(4099, 1000, 4001), (4100, 1024, 4032), (8200, 1224, 16100)])
def test_large_tiles_of_every_product(R, D, V, dt):
    """128 x 128 tiles for the logits, dx and dkernel alike: with tails along every axis, copied (4001 wide) and read where they lie (4032), in one piece
    and in several (16100)."""
    from aesrc2020_amd.losses import vocab_crossentropy, vocab_crossentropy_grad
    x, w, lab, b, dl = make(R, D, V, DT[dt], seed=R)
    want, bd = reference(x, w, lab, b, dl)
    loss, lse = vocab_crossentropy(x, w, lab, b, return_lse=True)
    check(loss, want[0], bd[0], "loss"); check(lse, want[1], bd[1], "lse")
    got = vocab_crossentropy_grad(dl, x, w, lab, lse, b)
    for g, wv, e, n in zip(got, want[2:], bd[2:], ("dx", "dkernel", "dbias")):
        check(g, wv, e, n)
    again = vocab_crossentropy_grad(dl, x, w, lab, lse, b)
    assert all(torch.equal(g, h) for g, h in zip(got, again))
