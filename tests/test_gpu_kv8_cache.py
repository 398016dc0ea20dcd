"""The 8-bit key / value cache on the GPU: the largest caches, scales and sizes of values at the ends of the range, appended chunks."""
import math

import pytest
import torch

from tests import _attn_ref as R
from tests.test_gpu_attention import DT, bounds, check, lens, make

pytestmark = pytest.mark.gpu


def test_more_blocks_than_one_row_of_a_launch():
    """4 x 2^28 + 64 frames of one narrow head: 2^24 + 4 blocks on each side (17 GB).  The frames all lie at one address."""
    from aesrc2020_amd.attention import EncoderCache8
    B, T, D = 4, (1 << 28) + 64, 8
    one = torch.tensor([1.0, -2.0, 3.0, 0.5, 448.0, 0.0, 7.0, -0.25], device="cuda").half()
    k = one.view(1, 1, 1, D).expand(B, T, 1, D)
    c = EncoderCache8(B, T, 1, D)
    c.store(k, -k, lens(T, T - 1, 0, 64))
    for y, s, v in ((c.k8, c.k_scale, one), (c.v8, c.v_scale, -one)):
        row = v.to(torch.float8_e4m3fn).view(torch.uint8).view(torch.int64)        # eight values: one word
        for b, n in enumerate((T, T - 1, 0, 64)):
            w = y[b, 0].view(torch.uint8).view(-1).view(torch.int64)
            assert (w[:n] == row).all() and (w[n:] == 0).all()
        assert (s == 1).all()
    assert c.lens.tolist() == [T, T - 1, 0, 64]
