"""Attention's forward where the operand types' range comes in: probabilities far below the largest, and large scores."""
import math

import pytest
import torch

from tests import _attn_ref as R
from tests.test_gpu_attention import DT, bounds, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("far", [8.3, 14.4, 19.6, 24.7])
@pytest.mark.parametrize("B,Tq,Tk", [(1, 1, 700), (2, 1, 5000), (1, 100, 1100), (1, 70, 9000)])
def test_a_key_without_a_value_takes_the_weight(B, Tq, Tk, far, dt):
    """One frame whose v is 0 (an attention sink) has 2^far times the weight of each other, which are alike (so that roundings of p do not cancel): the
    result is the others', to the operand type's rounding.  First, last, and in the middle of the frames."""
    from aesrc2020_amd.attention import EncoderCache8, cross_attention
    g = torch.Generator(device="cuda").manual_seed(int(far))
    H, D = 2, 32
    q = torch.zeros(B, Tq, H, D, device="cuda"); q[..., 0] = 4.0
    k = torch.zeros(B, Tk, H, D, device="cuda")
    v = 1.0 + 0.25 * torch.randn(B, Tk, H, D, generator=g, device="cuda")
    for at in (0, Tk // 2 + 3, Tk - 1):
        kk, vv = k.clone(), v.clone()
        kk[:, at, :, 0] = far * math.log(2) / 4.0
        vv[:, at] = 0.0
        a = [t.to(DT[dt]) for t in (q, kk, vv)]
        want = R.attend(*a, scale=1.0)
        check(cross_attention(*a, scale=1.0), want[0], bounds(*a, None, None, 1.0), "out", DT[dt])
        c = EncoderCache8(B, Tk, H, D)
        c.store(*a[1:])
        wide = [(y.float().double() * s.double().repeat_interleave(64, 2)[..., None])[:, :, :Tk].transpose(1, 2) for y, s in ((c.k8, c.k_scale), (c.v8, c.v_scale))]
        check(c.attend(a[0], scale=1.0), R.attend(a[0], *wide, scale=1.0)[0], bounds(a[0], *wide, None, None, 1.0), "cache", DT[dt])


def test_fp16_scores_that_step_by_sixteen():
    """Scores around 2^27 (in powers of two, where fp32 steps by 16) that grow from tile to tile: the last key has the weight, nothing is infinite."""
    from aesrc2020_amd.attention import cross_attention
    for Tq in (1, 80):
        for width in (32, 64, 128, 256):                           # what a wave, or a block, takes at a time
            for base in (2 ** 13 + 2 ** 3 * j for j in range(4)):
                q = torch.zeros(1, Tq, 1, 16, device="cuda", dtype=torch.float16); q[..., 0] = 16384.0; q[..., 1] = 16.0
                k = torch.zeros(1, 1100, 1, 16, device="cuda", dtype=torch.float16)
                k[0, :, 0, 0] = float(base)
                k[0, :, 0, 1] = torch.arange(1100, device="cuda").div(width, rounding_mode="floor").half()
                v = torch.ones(1, 1100, 1, 16, device="cuda", dtype=torch.float16)
                out, lse = cross_attention(q, k, v, scale=math.log(2), return_lse=True)
                # sums of weights of ones
                assert (out == 1).all() and torch.isfinite(lse).all(), (Tq, width, base)
