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


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("Tq", [1, 3])
def test_scores_of_no_size(Tq, dt):
    """A scale of 0, and keys so small that their scores' factor leaves fp32's range: every frame weighs the same, those behind the length nothing."""
    from aesrc2020_amd.attention import EncoderCache8
    q, k, v, _ = make(2, Tq, 150, 4, 2, 32, torch.float32, seed=9)
    kl = lens(150, 37)
    c = EncoderCache8(2, 150, 2, 32)
    for size, scale in ((1.0, 0.0), (2.0 ** -60, 0.0), (2.0 ** -125, 0.0), (2.0 ** 100, 0.0), (2.0 ** -120, 1e-20), (2.0 ** -125, 1.0)):
        c.store(k * size, v, kl)
        out = c.attend(q.to(DT[dt]), scale=scale)
        held = (c.v8.float() * c.v_scale.repeat_interleave(64, 2)[..., None])[:, :, :150].transpose(1, 2).double()
        for b, n in enumerate((150, 37)):
            want = held[b, :n].mean(0).repeat_interleave(2, 0).expand(Tq, 4, 32)
            # all p are 1 (or share one rounding), n + 3 fp32 sums of them and of v, the result's rounding
            lim = 2.0 ** -24 * (2 * n + 8) * held[b, :n].abs().mean(0).repeat_interleave(2, 0) + torch.finfo(DT[dt]).eps / 2 * want.abs()
            assert ((out[b].double() - want).abs() <= lim + (2.0 ** -25 if dt == "f16" else 0.0)).all(), (size, scale, b)


def test_a_scale_of_zero_makes_nothing_of_large_scores():
    """q . k of 2^120 on some keys, of -2^120 on others."""
    from aesrc2020_amd.attention import cross_attention
    g = torch.Generator(device="cuda").manual_seed(3)
    k = torch.ones(1, 70, 1, 16, device="cuda") * torch.where(torch.arange(70, device="cuda") % 3 == 0, -1.0, 1.0)[None, :, None, None]
    v = torch.randn(1, 70, 1, 16, generator=g, device="cuda")
    for n in (1, 50):
        out = cross_attention(torch.full((1, n, 1, 16), 2.0 ** 116, device="cuda"), k, v, scale=0.0)
        assert torch.allclose(out.double(), v.double().mean(1, keepdim=True).expand(1, n, 1, 16), rtol=0, atol=80 * 2.0 ** -23)


@pytest.mark.parametrize("Tk", [256, 1100])
def test_blocks_beyond_all_ratios(Tk):
    """fp16 queries over V blocks of 2^118 and 2^-38, in turn for every wave: columns that only the small blocks reach come out as 0, the others as infinities, none as NaN."""
    from aesrc2020_amd.attention import EncoderCache8
    q, k, v, _ = make(1, 3, Tk, 2, 1, 32, torch.float32, seed=Tk)
    big = (torch.arange(Tk, device="cuda") // 64 % 3 == 0)[None, :, None, None]
    v = torch.where(big, 2.0 ** 118, 2.0 ** -38) * (1 + v.abs())
    v[..., 8:] *= ~big
    c = EncoderCache8(1, Tk, 1, 32)
    c.store(k, v)
    out = c.attend(q.half())
    assert (out[..., 8:] == 0).all() and torch.isposinf(out[..., :8]).all()


def test_chunks_start_where_the_ones_before_end():
    """A gap would be attended to, whatever lies there: a new cache's memory, or another utterance's frames."""
    from aesrc2020_amd.attention import EncoderCache8
    _, k, v, _ = make(2, 1, 320, 2, 2, 16, torch.float32, seed=1)
    c = EncoderCache8(2, 320, 2, 16)
    for first in (64, 256):
        with pytest.raises(ValueError, match="never stored"):
            c.store(k[:, :64], v[:, :64], first=first)
    c.store(k[:, :100], v[:, :100]); c.store(k[:, 128:], v[:, 128:], first=128)
    assert c.lens.tolist() == [320, 320]
    c.store(k[:, :70], v[:, :70])                                  # the next utterances: what lies behind is the last ones'
    with pytest.raises(ValueError, match="never stored"):
        c.store(k[:, 192:], v[:, 192:], first=192)
    c.store(k[:, 64:128], v[:, 64:128], first=64)                  # a block again, with its later frames
    assert c.lens.tolist() == [128, 128] and c.stored == 128
    c.stored = 256                                                 # filled by other means
    c.store(k[:, 256:], v[:, 256:], first=256)


@pytest.mark.parametrize("dt", DT)
def test_chunks_are_one_store(dt):
    """Appended chunks of whole blocks hold and answer what one store does, in every type."""
    from aesrc2020_amd.attention import EncoderCache8
    q, k, v, _ = make(3, 2, 450, 4, 2, 40, DT[dt], seed=7)
    c, d = EncoderCache8(3, 450, 2, 40), EncoderCache8(3, 450, 2, 40)
    d.store(k, v, lens(450, 130, 64))
    c.store(k[:, :64], v[:, :64]); c.store(k[:, 64:192], v[:, 64:192], lens(128, 66, 0), first=64); c.store(k[:, 192:], v[:, 192:], lens(258, 0, 0), first=192)
    assert c.lens.tolist() == d.lens.tolist() == [450, 130, 64]
    for a, b in ((c.k8, d.k8), (c.v8, d.v8)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert torch.equal(c.k_scale, d.k_scale) and torch.equal(c.v_scale, d.v_scale) and torch.equal(c.attend(q), d.attend(q))
